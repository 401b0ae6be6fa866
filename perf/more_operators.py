"""The measured cases of sampled decoding with drafted tokens over caches in pages: a step's rows are normed and
rotated, attend over pages of 4-bit or f16 keys and values, their logits become probabilities, drafted tokens are
verified against those from given random numbers, and the kept rows are appended to the pages.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes a case's inputs on the device,
`run()` is one pass: the plain torch form, or with `own` the framework's calls; `exact()` is the same pass in 64 bits.
The shapes are those of the Whisper-shaped synthetic model (20 heads of 64, 448 positions, 51866 logits in rows of
51904), and generic ones with shared key heads, other head sizes and long caches.

A cache lies in pages of `page` positions.  A page holds, per key head, tiles of 32 positions; lane 16g + m (g < 4,
m < 16) of a wavefront finds what the matrix cores want of it in words of 8 values: word (c, u) of K the values
32c + 8g .. + 7 of position 16u + m, word (c, x) of V value 32c + 2m + x of the positions 16(e / 4) + 4g + e % 4,
e < 8.  4 bits: value (nibble - 8) * d, element e in nibble e / 2 + 4 (e % 2) of the word; a tile's K words (four words
of a lane next to each other, the last two where their number is no multiple of four), the f16 factors d of K
([g][c][e], for position 16(e / 4) + 4g + e % 4 and the values from 32c on), V's words and V's factors.  f16: 8 halfs for
the word, K [c][u][lane][e] and V [c][x][lane][e].
"""

import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
NONE = -1  # the pick of a row that the walk does not reach, or with nothing left
EPS = 1e-6  # of the norms


def listed():
    return [
        # One token's queries and keys of one sequence: the smallest call, between a decoder layer's projection and its attention.
        {"name": "norm_token", "kind": "norm", "batch": 1, "rows": 1, "heads": 20, "kv_heads": 20, "hd": 64, "rot": 64,
         "pairs": False, "norm": True, "tree": False, "longest": 448, "half": False, "half_out": False},
        # The rows of a batch of long prompts, f16, with shared key heads.
        {"name": "norm_prompt", "kind": "norm", "batch": 8, "rows": 1024, "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128,
         "pairs": False, "norm": True, "tree": False, "longest": 32768, "half": True, "half_out": True},
        # A decoding batch's tokens: a position each, normed, rotated and stored in 4 bits, queries on the way.
        {"name": "append_token", "kind": "append", "batch": 16, "rows": 1, "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128,
         "pairs": False, "norm": True, "path": False, "page": 64, "bits": 4, "longest": 32768, "half": False},
        # The kept paths of a batch's drafted tokens, rotated already, into f16 pages.
        {"name": "append_path", "kind": "append", "batch": 32, "rows": 61, "heads": 20, "kv_heads": 20, "hd": 64, "rot": 0,
         "pairs": False, "norm": False, "path": True, "page": 32, "bits": 16, "longest": 448, "half": False},
        # Long prompts into 4-bit pages: the largest call of the kind.
        {"name": "append_prompt", "kind": "append", "batch": 8, "rows": 1024, "heads": 32, "kv_heads": 8, "hd": 128, "rot": 128,
         "pairs": False, "norm": True, "path": False, "page": 256, "bits": 4, "longest": 32768, "half": True},
        # One new token of one sequence half way through its window.
        {"name": "attend_token", "kind": "attend", "batch": 1, "rows": 1, "heads": 20, "kv_heads": 20, "hd": 64, "page": 32,
         "bits": 4, "shortest": 224, "longest": 224, "half": False},
        # A decoding batch without drafts over caches of different lengths.
        {"name": "attend_decode", "kind": "attend", "batch": 32, "rows": 1, "heads": 32, "kv_heads": 8, "hd": 128, "page": 64,
         "bits": 4, "shortest": 1000, "longest": 8191, "half": True},
        # Trees of drafted tokens over long caches.
        {"name": "attend_tree", "kind": "attend", "batch": 8, "rows": 25, "heads": 32, "kv_heads": 8, "hd": 128, "page": 128,
         "bits": 4, "shortest": 24000, "longest": 32743, "half": True},
        # One row of logits of one sequence.
        {"name": "probs_token", "kind": "probs", "batch": 1, "rows": 1, "vocab": 51866, "ld": 51904, "half": False},
        # The rows of a batch's trees.
        {"name": "probs_tree", "kind": "probs", "batch": 16, "rows": 24, "vocab": 51866, "ld": 51904, "half": False},
        # One sequence's chain of drafted tokens without the drafts' probabilities (a known text).
        {"name": "sample_token", "kind": "sample", "batch": 1, "rows": 8, "vocab": 51866, "ld": 51904, "draft": False, "spread": 1},
        # A batch's trees with the drafts' probabilities.
        {"name": "sample_tree", "kind": "sample", "batch": 32, "rows": 24, "vocab": 51866, "ld": 51904, "draft": True, "spread": 7},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["norm", "append", "append", "attend", "attend", "attend", "probs", "sample"])
    half = rng.random() < 0.5
    if kind in ("probs", "sample"):
        vocab, batch = _spread(rng, 1000, 131072), _spread(rng, 1, 32)
        rows = _spread(rng, 1, max(1, min(64, (20 if kind == "probs" else 40) * 10**6 // (vocab * batch))))
        c = {"kind": kind, "batch": batch, "rows": rows, "vocab": vocab, "ld": vocab + rng.choice([0, 1, -vocab % 64])}
        return {**c, "half": half} if kind == "probs" else {**c, "draft": rng.random() < 0.6, "spread": rng.choice([1, 2, 7])}
    hd = rng.choice([64, 64, 128, 128, 32, 96] + ([80, 40] if kind == "norm" else []))
    kv_heads = rng.choice([20, 20, 16, 8, 5, 4, 2])
    heads = kv_heads * (1 if kv_heads == 20 else rng.choice([1, 1, 2, 3, 4, 8]))
    c = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "hd": hd, "half": half}
    if kind == "attend":
        bits = rng.choice([4, 4, 16])
        batch, rows = _spread(rng, 1, 24), _spread(rng, 1, 64)
        # Within the listed trees' cache values and products.
        most = min(32768, 268435456 // (batch * kv_heads * hd), 2 * 10**10 // (batch * rows * heads * hd))
        longest = rng.randint(0, _spread(rng, 16, max(17, most)))
        return {**c, "batch": batch, "rows": rows, "page": rng.choice([32, 64, 128, 256]), "bits": bits,
                "shortest": rng.randint(longest // 2, longest), "longest": longest}
    batch = _spread(rng, 1, 32)
    rows = _spread(rng, 1, max(1, min(1024, 4 * 10**7 // (batch * (heads + 2 * kv_heads) * hd))))
    c.update(batch=batch, rows=rows, rot=rng.choice([hd, hd, hd // 16 * 8]), pairs=rng.random() < 0.3, norm=rng.random() < 0.7)
    if kind == "norm":
        return {**c, "tree": rows <= 64 and rng.random() < 0.5, "longest": _spread(rng, 64, 32768), "half_out": half and rng.random() < 0.7}
    if rng.random() < 0.4:
        c.update(path=True, rows=min(rows, 64), rot=0, norm=False)
    else:
        c.update(path=False)
    return {**c, "page": rng.choice([32, 64, 128, 256]), "bits": rng.choice([4, 4, 16]), "longest": _spread(rng, 64, 32768)}


# ------------------------------------------------------------------------------------------ inputs


def _generator(seed, what):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000 * seed + what)
    return g


def _randn(seed, what, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=_generator(seed, what), device=DEV, dtype=dtype)


def _trees(rng, batch, rows, spread):
    """Per sequence: how many nodes it has and their parents, at most `spread` nodes before them."""
    count = rng.integers((rows + 1) // 2, rows + 1, batch)
    parents = np.zeros((batch, rows), np.int64)
    for i in range(1, rows):
        parents[:, i] = rng.integers(max(0, i - spread), i, batch)
    return count, parents


def _masks(parents):
    """The bits of every node and its ancestors, [batch][rows][words] 32-bit words."""
    batch, rows = parents.shape
    seen = np.zeros((batch, rows, 32 * ((rows + 31) // 32)), bool)
    for i in range(rows):
        if i:
            seen[:, i] = seen[np.arange(batch), parents[:, i]]
        seen[:, i, i] = True
    words = np.packbits(seen, axis=-1, bitorder="little").view(np.uint32)
    return np.ascontiguousarray(words).view(np.int32)


def _tile_words(c):
    """32-bit words of a tile: 32 positions of one key head."""
    return 9 * c["hd"] if c["bits"] == 4 else 32 * c["hd"]


def _pool(c, seed, pages):
    """A pool of pages as earlier tokens have left it."""
    shape = (pages, c["kv_heads"], c["page"] // 32, _tile_words(c))
    if c["bits"] == 16:
        return _randn(seed, 1, *shape, 2, dtype=torch.float16).view(torch.int32).view(shape)
    # Nibbles around the middle, as rounding gives them, and factors of either sign.
    g, hd = _generator(seed, 1), c["hd"]
    pool = torch.empty(shape, device=DEV, dtype=torch.int32)
    for at in range(0, pages, 2048):
        part = pool[at:at + 2048]
        a, b = (torch.randint(-2**31, 2**31, part.shape, generator=g, device=DEV, dtype=torch.int32) for _ in range(2))
        part.copy_((a & 0x77777777) + (b & 0x77777777))
        for first in (4 * hd, 8 * hd + hd // 2):
            d = torch.randn(*part.shape[:-1], hd, generator=g, device=DEV)
            d = torch.where(d > 0, 0.25, -0.25) * torch.exp(0.2 * d)
            part[..., first:first + hd // 2] = d.half().view(torch.int32)
    return pool


def _rope_table(positions, rot):
    """[positions][cos | sin] of rot / 2 angles."""
    angle = np.arange(positions)[:, None] * 10000.0 ** (-2.0 * np.arange(rot // 2) / rot)
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def _softmax(x):
    return torch.softmax(x, -1)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    s = {"kind": case["kind"], "case": case}
    batch, rows, kind = case["batch"], case["rows"], case["kind"]
    count, parents = _trees(rng, batch, rows, case.get("spread", 7))
    if kind in ("norm", "append") and not case.get("tree") and not case.get("path"):
        count[:] = rows  # consecutive tokens, all there
    s["count"], s["mask"] = dev(count.astype(np.int32)), dev(_masks(parents))
    if kind in ("norm", "append", "attend"):
        h, g, hd = case["heads"], case["kv_heads"], case["hd"]
        number = torch.float16 if case["half"] else torch.float32
        x = _randn(seed, 2, batch, rows, (h + 2 * g) * hd)  # the projections' rows [q | k | v]
        x[..., :h * hd] *= 2
        s["x"] = x.to(number)
    if kind in ("norm", "append"):
        if case["norm"]:
            s["q_gain"], s["k_gain"] = (1 + 0.1 * _randn(seed, 3 + i, hd) for i in range(2))
        n = rng.integers(0, max(1, case["longest"] - rows), batch)
        if case["rot"]:
            s["table"] = dev(_rope_table(int(n.max()) + rows, case["rot"]))
    if kind == "norm":
        s["n"] = dev(n.astype(np.int32))
        s["y"] = torch.zeros(batch, rows, (h + 2 * g) * hd, device=DEV, dtype=torch.float16 if case["half_out"] else torch.float32)
    elif kind in ("append", "attend"):
        if kind == "attend":
            n = rng.integers(case["shortest"], case["longest"] + 1, batch)
            n[0] = case["longest"]
            s["o"] = torch.zeros(batch, rows, h * hd, device=DEV, dtype=number)
        else:
            s["qo"] = torch.zeros(batch, rows, h * hd, device=DEV, dtype=torch.float16 if case["half"] else torch.float32)
            s["k"], s["v"] = (torch.zeros(batch, rows, g * hd, device=DEV, dtype=torch.float16) for _ in range(2))
            s["n_out"] = torch.zeros(batch, device=DEV, dtype=torch.int32)
            s["kept"] = s["count"]
            if case["path"]:
                # An accepted path of the tree: some nodes in order, at least the root.
                kept = 1 + rng.integers(0, count, batch) // 3
                path = np.full((batch, rows), -1, np.int32)
                for b in range(batch):
                    path[b, :kept[b]] = np.concatenate([[0], 1 + np.sort(rng.permutation(count[b] - 1)[:kept[b] - 1])])
                s["path"], s["kept"] = dev(path), dev(kept.astype(np.int32))
        s["n"] = dev(n.astype(np.int32))
        # The pages of each sequence, anywhere in the pool; those of an append alone, as the rest of the pool is not touched.
        first = n // case["page"] if kind == "append" else 0 * n
        used = (n + (rows if kind == "append" else 0) + case["page"] - 1) // case["page"]
        table = np.full((batch, max(1, int(used.max()))), -1, np.int32)
        ids = rng.permutation(max(1, int((used - first).sum())))
        at = 0
        for b in range(batch):
            table[b, first[b]:used[b]] = ids[at:at + used[b] - first[b]]
            at += used[b] - first[b]
        s["table_of_pages"], s["pages"] = dev(table), len(ids)
        s["pool"] = _pool(case, seed, len(ids))
        if kind == "append":  # where the plain form stores the values themselves
            s["stored"] = torch.zeros(2, len(ids) * case["page"] + 1, g * hd, device=DEV, dtype=torch.float16)
    elif kind == "probs":
        s["n"] = dev(np.zeros(batch, np.int32))
        s["temperature"] = dev(rng.uniform(0.2, 1.5, batch).astype(np.float32))
        s["logits"] = (4 * _randn(seed, 4, batch * rows, case["ld"])).to(torch.float16 if case["half"] else torch.float32)
        s["probs"] = torch.zeros(batch * rows, case["ld"], device=DEV)
    else:
        vocab, ld = case["vocab"], case["ld"]
        s["n"] = dev(np.zeros(batch, np.int32))
        s["u"] = torch.rand(batch, rows, generator=_generator(seed, 5), device=DEV)
        # A draft model's logits near the target's, with few likely ids; every node's token drawn from its parent's drafts.
        x = 10 * _randn(seed, 4, batch * rows, ld)
        x[:, vocab:] = -math.inf
        s["p"] = _softmax(x)
        x += _randn(seed, 6, batch * rows, ld)
        q = _softmax(x)
        of = (torch.from_numpy(parents).to(DEV) + rows * torch.arange(batch, device=DEV)[:, None]).view(-1)
        drawn = torch.cumsum(q, 1, out=x)
        at = torch.rand(batch * rows, generator=_generator(seed, 7), device=DEV) * drawn[of, vocab - 1]
        tokens = torch.cat([torch.searchsorted(drawn[of[i:i + 256]], at[i:i + 256, None]) for i in range(0, batch * rows, 256)])
        s["tokens"] = tokens.clamp(max=vocab - 1).view(batch, rows).int()
        s["q"] = q if case["draft"] else None
        s["picks"] = torch.zeros(batch, rows, device=DEV, dtype=torch.int32)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------- one pass


@functools.lru_cache(None)
def _gpu():
    import wavo_amd

    return wavo_amd.Gpu(0)


def _at(x):
    return None if x is None else x.data_ptr()


def _tree(s, masked=True):
    import wavo_amd

    return wavo_amd.Tree(s["case"]["batch"], s["case"]["rows"], _at(s["n"]), _at(s["count"]), _at(s.get("tokens")),
                         _at(s["mask"]) if masked else None, s["mask"][0].numel())


def _heads(s):
    import wavo_amd

    c, table = s["case"], s.get("table")
    return wavo_amd.Heads(c["heads"], c["kv_heads"], c["hd"], _at(s.get("q_gain")), _at(s.get("k_gain")), EPS, _at(table),
                          0 if table is None else len(table), c["rot"], c["pairs"])


def _pages(s):
    import wavo_amd

    c, table = s["case"], s["table_of_pages"]
    return wavo_amd.Pages(_at(s["pool"]), s["pages"], _at(table), table.shape[1], table.shape[1], c["page"],
                          wavo_amd.Q4_0 if c["bits"] == 4 else wavo_amd.F16, c["kv_heads"], c["hd"])


def run(s):
    return {"norm": _norm, "append": _append, "attend": _attend, "probs": _probs, "sample": _sample}[s["kind"]](s)


def _seen(s):
    """[batch][rows][rows] truth values: node i sees node j, both of them there."""
    c = s["case"]
    j = torch.arange(c["rows"], device=DEV)
    bits = (s["mask"][:, :, j // 32] >> (j % 32)) & 1
    there = j < s["count"][:, None]
    return (bits != 0) & there[:, :, None] & there[:, None, :], there


def _normed(c, x, gain):
    """Heads [..., hd] by their root mean square and gains."""
    return x if gain is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gain.to(x.dtype)


def _rotated(c, x, table, position):
    """The first `rot` values of every head [batch][rows][heads][hd] turned by their position's angles."""
    if not c["rot"]:
        return x
    half = c["rot"] // 2
    cos, sin = (t.to(x.dtype)[:, :, None] for t in table[position.clamp(max=len(table) - 1)].split(half, -1))
    a, b = (x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]) if c["pairs"] else (x[..., :half], x[..., half:c["rot"]])
    y = [a * cos - b * sin, b * cos + a * sin]
    y = torch.stack(y, -1).flatten(-2) if c["pairs"] else torch.cat(y, -1)
    return torch.cat([y, x[..., c["rot"]:]], -1)


def _norm(s):
    c = s["case"]
    batch, rows, h, g, hd = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["hd"]
    if own:
        d = (h + 2 * g) * hd
        _gpu().head_norm(_tree(s, c["tree"]), _heads(s), _at(s["x"]), d, _at(s["y"]), d, in16=c["half"], out16=c["half_out"])
        return s["y"]
    seen, there = _seen(s)
    j = torch.arange(rows, device=DEV)
    depth = (seen & (j < j[:, None])).sum(2) if c["tree"] else j.expand(batch, rows)
    x = s["x"].float().view(batch, rows, h + 2 * g, hd)
    parts = [(x[:, :, :h], s.get("q_gain")), (x[:, :, h:h + g], s.get("k_gain"))]
    y = [_rotated(c, _normed(c, p, gain), s.get("table"), s["n"][:, None] + depth) for p, gain in parts]
    y = torch.cat(y + [x[:, :, h + g:]], 2).view(batch, rows, -1)
    return torch.where(there[:, :, None], y, 0.0).to(s["y"].dtype)


def _in_4_bits(x):
    """f16 values as Q4_0 holds them: per 32 d = m / -8 of the one of largest magnitude, x / d to the nearest of -8 .. 7."""
    x = x.float().unflatten(-1, (-1, 32))
    top, bottom = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    d = (torch.where(top >= -bottom, top, bottom) / -8).half().float()
    q = torch.where(d != 0, torch.floor(x / d + 8.5).clamp(0, 15), 8.0)
    return ((q - 8) * d).flatten(-2).half()


def _append(s):
    c = s["case"]
    batch, rows, h, g, hd = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["hd"]
    turned = not c["path"]  # rows of a path have been normed and rotated where they attended
    if own:
        import wavo_amd

        x, size = _at(s["x"]), s["x"].element_size()
        heads = _heads(s) if turned else wavo_amd.Heads(h, g, hd)
        _gpu().page_append(_tree(s, False), heads, x if turned else None, x + size * h * hd, x + size * (h + g) * hd, s["x"].shape[-1],
                           _pages(s), path=_at(s.get("path")), kept=_at(s["kept"]), qo=_at(s["qo"]) if turned else None,
                           qo_stride=h * hd, n_out=_at(s["n_out"]), in16=c["half"], out16=c["half"])
        stored = wavo_amd.Tree(batch, rows, _at(s["n"]), _at(s["kept"]))
        _gpu().page_read(stored, _pages(s), _at(s["k"]), _at(s["v"]), g * hd, out16=True)
        return {"k": s["k"], "v": s["v"], "n": s["n_out"], **({"q": s["qo"]} if turned else {})}
    i = torch.arange(rows, device=DEV)
    there = i < s["kept"][:, None]
    row = s["path"].clamp(min=0).long() if c["path"] else i.expand(batch, rows)
    x = s["x"].gather(1, row[:, :, None].expand(-1, -1, s["x"].shape[-1])).view(batch, rows, h + 2 * g, hd)
    position = s["n"][:, None] + i
    # Keys in 64 bits: 4 bits' borders are near.
    k = _rotated(c, _normed(c, x[:, :, h:h + g].double(), s.get("k_gain")), s.get("table"), position) if turned else x[:, :, h:h + g]
    new = [t.half().reshape(batch, rows, g * hd) for t in (k, x[:, :, h + g:])]
    if c["bits"] == 4:
        new = [_in_4_bits(t) for t in new]
    page = s["table_of_pages"].gather(1, (position // c["page"]).clamp(max=s["table_of_pages"].shape[1] - 1).long())
    place = torch.where(there, page * c["page"] + position % c["page"], s["pages"] * c["page"])
    s["stored"][0, place], s["stored"][1, place] = new[0], new[1]
    k, v = (torch.where(there[:, :, None], t[place], 0.0) for t in s["stored"])
    out = {"k": k, "v": v, "n": s["n"] + s["kept"]}
    if turned:
        q = _rotated(c, _normed(c, x[:, :, :h].float(), s.get("q_gain")), s.get("table"), position)
        out["q"] = torch.where(there[:, :, None], q.reshape(batch, rows, h * hd), 0.0).to(s["qo"].dtype)
    return out


def _values(c, words):
    """Tiles [..., words] as keys and values [..., 32, hd] (see above)."""
    hd, chunks, shape = c["hd"], c["hd"] // 32, words.shape[:-1]
    if c["bits"] == 16:
        k, v = words.view(torch.float16).view(*shape, 2, chunks, 2, 4, 16, 8).unbind(-6)  # [c][u or x][g][m][e]
        k = k.movedim((-4, -2, -5, -3, -1), (-5, -4, -3, -2, -1))
        v = v.unflatten(-1, (2, 4)).movedim((-2, -4, -1, -6, -3, -5), (-6, -5, -4, -3, -2, -1))
        return k.reshape(*shape, 32, hd).float(), v.reshape(*shape, 32, hd).float()
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=DEV, dtype=torch.int32)
    got = []
    for part in words.split(9 * hd // 2, -1):
        w, whole = part[..., :4 * hd], 256 * (2 * chunks // 4)
        lanes = w[..., :whole].reshape(*shape, -1, 64, 4).transpose(-3, -2).reshape(*shape, 64, -1)
        w = torch.cat([lanes, w[..., whole:].reshape(*shape, 64, -1)], -1).view(*shape, 4, 16, chunks, 2)
        w = (w[..., None] >> shifts) & 15  # [g][m][c][u or x][e]
        d = part[..., 4 * hd:].contiguous().view(torch.float16).view(*shape, 4, chunks, 2, 4)  # [g][c][u][r]
        d = d.movedim((-2, -4, -1, -3), (-4, -3, -2, -1)).reshape(*shape, 32, chunks, 1).float()
        if not got:
            w = w.movedim((-2, -4, -3, -5, -1), (-5, -4, -3, -2, -1))
        else:
            w = w.unflatten(-1, (2, 4)).movedim((-2, -6, -1, -4, -5, -3), (-6, -5, -4, -3, -2, -1))
        got.append(((w.reshape(*shape, 32, chunks, 32) - 8) * d).view(*shape, 32, hd))
    return got


def _attend(s):
    c = s["case"]
    batch, rows, h, g, hd = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["hd"]
    if own:
        x, size = _at(s["x"]), s["x"].element_size()
        _gpu().page_attend(_tree(s), x, x + size * h * hd, x + size * (h + g) * hd, s["x"].shape[-1], _pages(s), _at(s["o"]), h,
                           in16=c["half"], out16=c["half"])
        return s["o"]
    K, V = _values(c, s["pool"][s["table_of_pages"].clamp(min=0).long()].transpose(1, 2))  # [batch][key head][page][tile][32][hd]
    K, V = (t.reshape(batch, g, -1, hd) for t in (K, V))
    there_keys = torch.arange(K.shape[2], device=DEV) < s["n"][:, None]
    seen, there = _seen(s)
    # A node's keys and values as f16.
    k, v = s["x"][..., h * hd:].half().float().view(batch, rows, 2, g, hd).permute(2, 0, 3, 1, 4)
    K, V = torch.cat([K, k], 2), torch.cat([V, v], 2)
    visible = torch.cat([there_keys[:, None, :].expand(batch, rows, -1), seen], 2)
    q = s["x"][..., :h * hd].float().view(batch, rows, g, h // g, hd).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q.reshape(batch, g, h // g * rows, hd), K.transpose(2, 3)) / math.sqrt(hd)
    score = torch.where(visible[:, None, None], score.view(batch, g, h // g, rows, -1), -math.inf)
    some = visible.any(2)[:, None, None, :, None]
    p = torch.exp(score - torch.where(some, score.amax(-1, keepdim=True), 0.0))
    o = torch.matmul(p.view(batch, g, h // g * rows, -1), V).view(batch, g, h // g, rows, hd)
    o = torch.where(some, o / p.sum(-1, keepdim=True), 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, rows, h * hd)
    return torch.where(there[:, :, None], o, 0.0).to(s["o"].dtype)


def _probs(s):
    c = s["case"]
    batch, rows, vocab = c["batch"], c["rows"], c["vocab"]
    if own:
        _gpu().logit_probs(_tree(s), _at(s["logits"]), _at(s["probs"]), vocab, c["ld"], c["ld"], temperature=_at(s["temperature"]),
                           half=c["half"])
        return s["probs"]
    there = _seen(s)[1].reshape(-1)
    x = s["logits"][:, :vocab].float()
    p = torch.exp((x - x.amax(1, keepdim=True)) / s["temperature"].repeat_interleave(rows)[:, None])
    out = torch.zeros_like(s["probs"])
    out[:, :vocab] = torch.where(there[:, None], p / p.sum(1, keepdim=True), 0.0)
    return out


def _sample(s):
    c = s["case"]
    batch, rows, vocab = c["batch"], c["rows"], c["vocab"]
    if own:
        _gpu().tree_sample(_tree(s), _at(s["p"]), _at(s["q"]), vocab, c["ld"], _at(s["u"]), _at(s["picks"]))
        return s["picks"]
    # Node by node; 64 bits, as sums of so many values are compared with random numbers.
    seen, there = _seen(s)
    b, i = torch.arange(batch, device=DEV), torch.arange(rows, device=DEV)
    parent = torch.where(seen & (i < i[:, None]), i, -1).amax(2)
    p = s["p"].view(batch, rows, -1)[..., :vocab]
    q = None if s["q"] is None else s["q"].view(batch, rows, -1)[..., :vocab]
    tokens, u = s["tokens"].long(), s["u"].double()
    at = torch.zeros(batch, device=DEV, dtype=torch.int64)
    w, total = p[:, 0].double(), torch.ones(batch, device=DEV, dtype=torch.float64)
    picks = torch.full((batch, rows), NONE, device=DEV, dtype=torch.int32)
    for node in range(1, rows):
        x = tokens[:, node]
        mine = w[b, x]
        tested = (parent[:, node] == at) & there[:, node] & (total > 0)
        hit = tested & (u[:, node] * (1.0 if q is None else q[b, at, x].double()) * total < mine)
        miss = tested & ~hit
        if q is None:
            left = w.clone()
            left[b, x] = 0.0
            rest = total - mine
        else:
            left = (w / total[:, None] - q[b, at].double()).clamp(min=0.0)
            rest = left.sum(1)
        picks[b, at] = torch.where(hit, x.int(), picks[b, at])
        w = torch.where(hit[:, None], p[:, node].double(), torch.where(miss[:, None], left, w))
        total = torch.where(hit, 1.0, torch.where(miss, rest, total))
        at = torch.where(hit, node, at)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, p[b, at].double())
    sums = torch.cumsum(w, 1)
    found = sums > u[:, :1] * sums[:, -1:]
    picks[b, at] = torch.where(found.any(1), found.int().argmax(1), NONE).int()
    return torch.where(there, picks, 0)


# --------------------------------------------------------------------------------------------- work


def work(case):
    batch, rows, kind = case["batch"], case["rows"], case["kind"]
    nodes = batch * (rows + (rows + 1) // 2) / 2  # the nodes that are there, on average
    if kind == "probs":
        return {"bytes": nodes * case["vocab"] * (6 if case["half"] else 8), "flops": 4.0 * nodes * case["vocab"]}
    if kind == "sample":  # the last row of the walk, of the target and of the drafts
        return {"bytes": 4.0 * batch * case["vocab"] * (2 if case["draft"] else 1), "flops": 4.0 * batch * case["vocab"]}
    h, g, hd, size = case["heads"], case["kv_heads"], case["hd"], 2 if case["half"] else 4
    cached = 9 / 16 if case.get("bits") == 4 else 2.0  # bytes of a value
    if kind == "norm":
        nodes = nodes if case["tree"] else batch * rows
        return {"bytes": nodes * (h + 2 * g) * hd * (size + (2.0 if case["half_out"] else 4.0)), "flops": 10.0 * nodes * (h + g) * hd}
    if kind == "append":
        nodes = nodes / 6 if case["path"] else batch * rows
        moved = 2 * g * hd * (size + 2 * cached + 2) + (0 if case["path"] else 2 * h * hd * size)  # in, stored, read, out
        return {"bytes": nodes * moved, "flops": 20.0 * nodes * g * hd}
    keys = (case["shortest"] + case["longest"]) / 2
    return {"bytes": 2.0 * batch * keys * g * hd * cached + size * nodes * 2 * (h + g) * hd,
            "flops": 4.0 * nodes * (keys + min(rows, 8)) * h * hd}


# ----------------------------------------------------------------------------------- 64-bit passes


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend, "probs": _exact_probs, "sample": _exact_sample}[case["kind"]](s)


def _sees(mask, i, j):
    return (int(mask[i, j // 32]) >> (j % 32)) & 1


def _exact_turn(s, x, gain, position):
    """Heads x [rows][heads][hd] of positions [rows]: normed, and each pair as a complex number times another."""
    c = s["case"]
    x = x.double()
    if gain is not None:
        x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / c["hd"] + EPS) * gain.double()
    if c["rot"]:
        half = c["rot"] // 2
        t = s["table"][position].double()
        turn = torch.complex(t[:, :half], t[:, half:])[:, None]
        of = torch.arange(c["rot"], device=DEV).view(half, 2) if c["pairs"] else torch.arange(c["rot"], device=DEV).view(2, half).T
        z = torch.complex(x[..., of[:, 0]], x[..., of[:, 1]]) * turn
        x = x.clone()
        x[..., of[:, 0]], x[..., of[:, 1]] = z.real, z.imag
    return x


def _exact_norm(s):
    c = s["case"]
    h, g, hd = c["heads"], c["kv_heads"], c["hd"]
    out = torch.zeros(s["y"].shape, device=DEV, dtype=torch.float64)
    for b in range(c["batch"]):
        count, mask = int(s["count"][b]), s["mask"][b].cpu().numpy()
        depth = [sum(_sees(mask, i, j) for j in range(i)) if c["tree"] else i for i in range(count)]
        position = int(s["n"][b]) + torch.tensor(depth, device=DEV)
        x = s["x"][b, :count].view(count, -1, hd)
        q, k = _exact_turn(s, x[:, :h], s.get("q_gain"), position), _exact_turn(s, x[:, h:h + g], s.get("k_gain"), position)
        out[b, :count] = torch.cat([q, k, x[:, h + g:].double()], 1).view(count, -1)
    return out


def _exact_append(s):
    c = s["case"]
    h, g, hd = c["heads"], c["kv_heads"], c["hd"]
    out = {"k": torch.zeros(s["k"].shape, device=DEV, dtype=torch.float64), "v": torch.zeros(s["v"].shape, device=DEV, dtype=torch.float64), "n": None}
    if not c["path"]:
        out["q"] = torch.zeros(s["qo"].shape, device=DEV, dtype=torch.float64)
    for b in range(c["batch"]):
        kept = int(s["kept"][b])
        rows = s["path"][b, :kept].long() if c["path"] else torch.arange(kept, device=DEV)
        position = int(s["n"][b]) + torch.arange(kept, device=DEV)
        x = s["x"][b, rows].view(kept, -1, hd)
        k, v = x[:, h:h + g].double(), x[:, h + g:].double()
        if not c["path"]:
            k = _exact_turn(s, k, s.get("k_gain"), position)
            out["q"][b, :kept] = _exact_turn(s, x[:, :h], s.get("q_gain"), position).view(kept, -1)
        for name, t in (("k", k), ("v", v)):
            t = t.half().double()
            if c["bits"] == 4:
                blocks = t.reshape(-1, 32)
                size = blocks.abs().amax(1, keepdim=True)
                positive = (blocks == size).any(1, keepdim=True)
                d = (torch.where(positive, size, -size) / -8).half().double()
                steps = torch.where(d == 0, 0.0, blocks / torch.where(d == 0, 1.0, d))
                t = torch.clamp(torch.floor(steps + 0.5), -8, 7) * d
            out[name][b, :kept] = t.reshape(kept, -1)
    return out


def _exact_attend(s):
    """Sequence by sequence, every value looked up by its own word and place; softmax(q.k / sqrt(hd)).v."""
    c = s["case"]
    h, g, hd, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    chunks, words = hd // 32, _tile_words(c)
    pos, dim = np.arange(32)[:, None], np.arange(hd)[None, :]
    group = pos % 16 // 4
    # Lane, word and element of a key and of a value, and where their factors stand.
    kl, kt, ke = 16 * (dim % 32 // 8) + pos % 16, 2 * (dim // 32) + pos // 16, dim % 8 + 0 * pos
    vl, vt, ve = 16 * group + dim % 32 // 2, 2 * (dim // 32) + dim % 2 + 0 * pos, 4 * (pos // 16) + pos % 4 + 0 * dim
    factor = (group * chunks + dim // 32) * 8 + 4 * (pos // 16) + pos % 4

    def read(tiles, lane, t, e, first):
        if c["bits"] == 16:
            at = torch.from_numpy(2 * first + (t * 64 + lane) * 8 + e).to(DEV)
            return tiles.view(torch.float16)[:, at.view(-1)].double().view(-1, 32, hd)
        whole = 2 * chunks // 4 * 4
        word = np.where(t < whole, t // 4 * 256 + lane * 4 + t % 4, whole * 64 + lane * 2 + t - whole)
        at, shift = (torch.from_numpy(a).to(DEV).view(-1) for a in (first + word, 4 * (e // 2 + 4 * (e % 2))))
        d = tiles.view(torch.float16)[:, torch.from_numpy(2 * (first + 4 * hd) + factor).to(DEV).view(-1)].double()
        return ((((tiles[:, at] >> shift) & 15) - 8) * d).view(-1, 32, hd)

    out = torch.zeros(s["o"].shape, device=DEV, dtype=torch.float64)
    for b in range(c["batch"]):
        n, count = int(s["n"][b]), int(s["count"][b])
        mask = s["mask"][b].cpu().numpy()
        hidden = torch.tensor([[not _sees(mask, i, j) for j in range(count)] for i in range(count)], device=DEV)
        x = s["x"][b, :count]
        nk, nv = x[:, h * hd:].half().double().reshape(count, 2, g, hd).unbind(1)
        q = x[:, :h * hd].double().reshape(count, h, hd)
        pages = s["table_of_pages"][b, :(n + page - 1) // page].long()
        for of in range(g):
            tiles = s["pool"][pages, of].reshape(-1, words)
            k = torch.cat([read(tiles, kl, kt, ke, 0).view(-1, hd)[:n], nk[:, of]])
            v = torch.cat([read(tiles, vl, vt, ve, words // 2).view(-1, hd)[:n], nv[:, of]])
            for head in range(of * (h // g), (of + 1) * (h // g)):
                t = q[:, head] @ k.T / hd**0.5
                t[:, n:].masked_fill_(hidden, -math.inf)
                out[b, :count, head * hd:(head + 1) * hd] = torch.softmax(t, 1) @ v
    return out


def _exact_probs(s):
    c = s["case"]
    out = torch.zeros(s["probs"].shape, device=DEV, dtype=torch.float64)
    for b in range(c["batch"]):
        at = slice(b * c["rows"], b * c["rows"] + int(s["count"][b]))
        out[at, :c["vocab"]] = torch.softmax(s["logits"][at, :c["vocab"]].double() / float(s["temperature"][b]), 1)
    return out


def _exact_sample(s):
    return None  # whole numbers
