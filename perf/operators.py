"""The measured cases of a decoder step over drafted tokens: one pass reads a tree of drafted tokens per
sequence, attends from every one of them, applies the requests' rules to their logits, and keeps the path
that the model agrees with.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes a case's inputs on the
device, `run()` is one pass: the plain torch form, or with `own` the framework's calls; `exact()` is the same
pass in 64 bits.  The shapes are those of the Whisper-shaped synthetic model (20 heads of 64, 448 positions,
1500 encoder frames, 51866 logits in rows of 51904), and generic ones with shared key heads, other head sizes
and long caches.

A step's data: `n[b]` committed tokens per sequence, whose keys and values lie in a cache of `cols` positions
(f16 pairs, K transposed: pair i of position j at word i*cols + j, then V by position), and up to `rows`
drafted tokens, the nodes, of which `count[b]` are there.  Bit j of node i's mask: node j is i or one of its
ancestors, so that i sees it; node 0 is the root, the token picked last.
"""

import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
NONE = -1  # the pick of a row with nothing left


def listed():
    return [
        # One new token of one sequence half way through its window: the smallest call, a decoder layer's step.
        {"name": "attend_token", "kind": "attend", "batch": 1, "rows": 1, "heads": 20, "kv_heads": 20, "hd": 64,
         "cols": 448, "shortest": 224, "longest": 224, "half": False, "cross": False},
        # A tree of drafted tokens over a nearly full window of one sequence.
        {"name": "attend_tree", "kind": "attend", "batch": 1, "rows": 16, "heads": 20, "kv_heads": 20, "hd": 64,
         "cols": 448, "shortest": 391, "longest": 391, "half": False, "cross": False},
        # The drafted tokens of four sequences over their encoder frames: cross attention, no node sees another.
        {"name": "attend_frames", "kind": "attend", "batch": 4, "rows": 13, "heads": 20, "kv_heads": 20, "hd": 64,
         "cols": 1500, "shortest": 1100, "longest": 1500, "half": False, "cross": True},
        # A batch of requests of different lengths with large trees, f16 rows as between layers.
        {"name": "attend_batch", "kind": "attend", "batch": 16, "rows": 61, "heads": 20, "kv_heads": 20, "hd": 64,
         "cols": 448, "shortest": 37, "longest": 448, "half": True, "cross": False},
        # Long caches with four query heads to a key head.
        {"name": "attend_long", "kind": "attend", "batch": 4, "rows": 25, "heads": 32, "kv_heads": 8, "hd": 128,
         "cols": 32768, "shortest": 24000, "longest": 32743, "half": True, "cross": False},
        # One row of logits of one sequence, every rule on.
        {"name": "rules_token", "kind": "rules", "batch": 1, "rows": 1, "vocab": 51866, "ld": 51904, "half": False,
         "history": 224, "biases": 40, "grammar": True},
        # A decoding batch without drafts or grammar: penalties and biases alone.
        {"name": "rules_decode", "kind": "rules", "batch": 48, "rows": 1, "vocab": 51866, "ld": 51904, "half": False,
         "history": 448, "biases": 100, "grammar": False},
        # The nodes of a batch, each with its own grammar state.
        {"name": "rules_tree", "kind": "rules", "batch": 16, "rows": 24, "vocab": 51866, "ld": 51904, "half": False,
         "history": 448, "biases": 100, "grammar": True},
        # Large trees over a large vocabulary of odd size after long texts, f16 logits.
        {"name": "rules_large", "kind": "rules", "batch": 8, "rows": 61, "vocab": 131071, "ld": 131072, "half": True,
         "history": 16000, "biases": 1000, "grammar": True},
        # One sequence's tree: the path that holds and its keys and values into four layers' caches.
        {"name": "accept_tree", "kind": "accept", "batch": 1, "rows": 16, "layers": 4, "d": 1280, "cols": 448,
         "kept": 4, "half": False},
        # The same for a batch with large trees, and long paths.
        {"name": "accept_batch", "kind": "accept", "batch": 32, "rows": 61, "layers": 4, "d": 1280, "cols": 448,
         "kept": 9, "half": False},
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "rules", "rules", "accept"])
    half = rng.random() < 0.5
    if kind == "attend":
        cross = rng.random() < 0.2
        hd = rng.choice([64, 64, 64, 128, 128, 40, 80, 100])
        kv_heads = rng.choice([20, 20, 16, 8, 5, 4, 2])
        heads = kv_heads * (1 if kv_heads == 20 else rng.choice([1, 1, 2, 3, 4, 8]))
        batch, rows = _spread(rng, 1, 24), _spread(rng, 1, 64)
        # Within the listed long case's cache bytes and products.
        most = min(32768, 134217728 // (batch * kv_heads * hd), 12 * 10**9 // (batch * rows * heads * hd))
        cols = _spread(rng, 16, max(17, most))
        longest = rng.randint(0 if not cross else 1, cols)
        return {"kind": kind, "batch": batch, "rows": rows, "heads": heads, "kv_heads": kv_heads, "hd": hd, "cols": cols,
                "shortest": rng.randint(longest // 2, longest), "longest": longest, "half": half, "cross": cross}
    if kind == "rules":
        vocab = _spread(rng, 1000, 131072)
        batch = _spread(rng, 1, 64)
        rows = _spread(rng, 1, max(1, min(64, 60000000 // (vocab * batch))))
        return {"kind": kind, "batch": batch, "rows": rows, "vocab": vocab, "ld": vocab + rng.choice([0, 1, -vocab % 64]),
                "half": half, "history": _spread(rng, 1, 16000), "biases": rng.choice([0, _spread(rng, 1, 1000)]),
                "grammar": rng.random() < 0.6}
    rows = _spread(rng, 1, 64)
    return {"kind": kind, "batch": _spread(rng, 1, 32), "rows": rows, "layers": rng.randint(1, 4),
            "d": 4 * _spread(rng, 16, 320), "cols": _spread(rng, 64, 448), "kept": rng.randint(1, max(1, rows // 2)), "half": half}


# ------------------------------------------------------------------------------------------ inputs


def _randn(seed, what, *shape, dtype=torch.float32):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000 * seed + what)
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _trees(rng, batch, rows, kept):
    """Per sequence: how many nodes it has, their parents, and a chain of `kept` nodes from the root."""
    count = rng.integers(max(kept, (rows + 1) // 2), rows + 1, batch)
    parents = np.zeros((batch, rows), np.int64)
    chains = []
    for b in range(batch):
        for i in range(1, rows):
            parents[b, i] = rng.integers(max(0, i - 7), i)
        chain = np.concatenate([[0], 1 + np.sort(rng.permutation(count[b] - 1)[:kept - 1])]).astype(np.int64)
        parents[b, chain[1:]] = chain[:-1]
        chains.append(chain)
    return count, parents, chains


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


def _texts(rng, vocab, *shape):
    """Token ids of a text: few frequent ones, many rare ones, so that some come again."""
    return np.minimum(np.floor(vocab ** rng.random(shape)), vocab - 1).astype(np.int32)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
    s = {"kind": case["kind"], "case": case}
    batch, rows = case["batch"], case["rows"]
    number = torch.float16 if case["half"] else torch.float32
    count, parents, chains = _trees(rng, batch, rows, case.get("kept", 1))
    s["count"], s["mask"] = dev(count.astype(np.int32)), dev(_masks(parents))
    if case["kind"] == "attend":
        h, g, hd, cols = case["heads"], case["kv_heads"], case["hd"], case["cols"]
        n = rng.integers(case["shortest"], case["longest"] + 1, batch)
        n[0] = case["longest"]
        s["n"] = dev(n.astype(np.int32))
        s["kv"] = _randn(seed, 1, batch, 2 * cols * g * hd, dtype=torch.float16).view(torch.int32)
        # The projections' rows [q | k | v] of every node; cross attention has q alone.  Queries large enough for
        # a few keys to matter more than the others.
        x = _randn(seed, 2, batch, rows, h * hd if case["cross"] else (h + 2 * g) * hd)
        x[..., :h * hd] *= 2
        s["x"] = x.to(number)
        s["o"] = torch.zeros(batch, rows, h * hd, device=DEV, dtype=number)
    elif case["kind"] == "rules":
        vocab, words = case["vocab"], (case["vocab"] + 31) // 32
        n = rng.integers(case["history"] // 2, case["history"] + 1, batch)
        s["n"] = dev(n.astype(np.int32))
        s["history"] = dev(_texts(rng, vocab, batch, case["history"]))
        s["tokens"] = dev(_texts(rng, vocab, batch, rows))
        # Repetition, frequency and presence penalties of every request.
        s["penalty"] = dev(np.stack([rng.uniform(1.0, 1.5, batch), rng.uniform(0, 0.5, batch), rng.uniform(0, 0.5, batch)], 1).astype(np.float32))
        start = np.concatenate([[0], np.cumsum(rng.integers(case["biases"] // 2, case["biases"] + 1, batch))])
        s["bias_start"] = dev(start.astype(np.int32))
        s["bias_id"] = dev(rng.integers(0, vocab, max(1, start[-1])).astype(np.int32))
        s["bias"] = dev(rng.normal(0, 3, max(1, start[-1])).astype(np.float32))
        s["biases"] = int(start[-1])
        g = torch.Generator(device=DEV)
        g.manual_seed(1000 * seed + 3)
        # A grammar allows half of the ids, a few, or one; the words' bits past the vocabulary are anything.
        allow = torch.randint(-2**31, 2**31, (batch * rows, words), generator=g, device=DEV, dtype=torch.int64).int()
        rare = torch.rand(batch * rows, words, generator=g, device=DEV) < 0.9
        s["allow"] = torch.where(rare & (torch.arange(batch * rows, device=DEV) % 3 == 1)[:, None], 0, allow) if case["grammar"] else None
        s["logits"] = (4 * _randn(seed, 4, batch * rows, case["ld"])).to(number)
        s["out"] = torch.zeros(batch * rows, case["ld"], device=DEV, dtype=number)
        s["pick"] = torch.zeros(batch * rows, device=DEV, dtype=torch.int32)
        s["logprob"] = torch.zeros(batch * rows, device=DEV)
    else:
        layers, d, cols = case["layers"], case["d"], case["cols"]
        n = rng.integers(0, cols - case["kept"] + 1, batch)
        tokens, picks = _texts(rng, 51866, batch, rows), _texts(rng, 51866, batch, rows)
        for b, chain in enumerate(chains):
            tokens[b, chain[1:]] = picks[b, chain[:-1]]
        s["n"], s["tokens"], s["picks"] = dev(n.astype(np.int32)), dev(tokens), dev(picks)
        s["history"] = dev(_texts(rng, 51866, batch, cols))
        s["x"] = _randn(seed, 2, layers, batch, rows, 3 * d).to(number)  # the layers' [q | k | v] rows
        s["kv"] = _randn(seed, 1, layers, batch, 2 * cols * d, dtype=torch.float16).view(torch.int32)
        s["path"] = torch.zeros(batch, rows, device=DEV, dtype=torch.int32)
        s["kept"], s["next"], s["n_out"] = (torch.zeros(batch, device=DEV, dtype=torch.int32) for _ in range(3))
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------- one pass


@functools.lru_cache(None)
def _gpu():
    import wavo_amd

    return wavo_amd.Gpu(0)


def _tree(s, masked=True):
    import wavo_amd

    at = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    return wavo_amd.Tree(s["case"]["batch"], s["case"]["rows"], s["n"].data_ptr(), s["count"].data_ptr(), at(s.get("tokens")),
                         s["mask"].data_ptr() if masked else None, s["mask"][0].numel())


def run(s):
    return {"attend": _attend, "rules": _rules, "accept": _accept}[s["kind"]](s)


def _seen(s):
    """[batch][rows][rows] truth values: node i sees node j, both of them there."""
    c = s["case"]
    j = torch.arange(c["rows"], device=DEV)
    bits = (s["mask"][:, :, j // 32] >> (j % 32)) & 1
    there = j < s["count"][:, None]
    return (bits != 0) & there[:, :, None] & there[:, None, :], there


def _attend(s):
    c = s["case"]
    batch, rows, h, g, hd, cols = c["batch"], c["rows"], c["heads"], c["kv_heads"], c["hd"], c["cols"]
    if own:
        x, size, d = s["x"].data_ptr(), s["x"].element_size(), g * hd
        k = None if c["cross"] else x + size * h * hd
        v = None if c["cross"] else x + size * (h * hd + d)
        _gpu().tree_attend(_tree(s, not c["cross"]), x, k, v, s["x"].shape[-1], s["kv"].data_ptr(), cols * d, cols,
                           s["o"].data_ptr(), h, g, hd, in16=c["half"], out16=c["half"])
        return s["o"]
    pairs = s["kv"].view(torch.float16)
    K = pairs[:, :cols * g * hd].view(batch, g, hd // 2, cols, 2).permute(0, 1, 3, 2, 4).reshape(batch, g, cols, hd).float()
    V = pairs[:, cols * g * hd:].view(batch, cols, g, hd).transpose(1, 2).float()
    committed = torch.arange(cols, device=DEV) < s["n"][:, None]
    seen, there = _seen(s)
    visible = committed[:, None, :].expand(batch, rows, cols)
    q = s["x"][..., :h * hd].float().view(batch, rows, g, h // g, hd).permute(0, 2, 3, 1, 4)
    if not c["cross"]:
        # A node's keys and values as the cache will hold them.
        k, v = s["x"][..., h * hd:].half().float().view(batch, rows, 2, g, hd).permute(2, 0, 3, 1, 4)
        K, V = torch.cat([K, k], 2), torch.cat([V, v], 2)
        visible = torch.cat([visible, seen], 2)
    V = torch.where(visible.any(1)[:, None, :, None], V, 0.0)
    score = torch.matmul(q.reshape(batch, g, h // g * rows, hd), K.transpose(2, 3)) / math.sqrt(hd)
    score = torch.where(visible[:, None, None], score.view(batch, g, h // g, rows, -1), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(visible.any(2)[:, None, None, :, None], top, 0.0))
    o = torch.matmul(p.view(batch, g, h // g * rows, -1), V).view(batch, g, h // g, rows, hd)
    total = p.sum(-1, keepdim=True)
    o = torch.where(visible.any(2)[:, None, None, :, None], o / total, 0.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, rows, h * hd)
    return torch.where(there[:, :, None], o, 0.0).to(s["o"].dtype)


def _rules(s):
    c = s["case"]
    batch, rows, vocab, ld = c["batch"], c["rows"], c["vocab"], c["ld"]
    if own:
        import wavo_amd

        rules = wavo_amd.Rules(penalty=s["penalty"].data_ptr(), history=s["history"].data_ptr(), history_cols=c["history"],
                               bias_start=s["bias_start"].data_ptr(), bias_id=s["bias_id"].data_ptr(), bias=s["bias"].data_ptr(),
                               bias_len=s["biases"], allow=s["allow"].data_ptr() if c["grammar"] else None)
        _gpu().logit_rules(_tree(s), rules, s["logits"].data_ptr(), s["out"].data_ptr(), vocab, ld, half=c["half"],
                           pick=s["pick"].data_ptr(), logprob=s["logprob"].data_ptr())
        return s["out"], s["pick"], s["logprob"]
    seen, there = _seen(s)
    x = s["logits"][:, :vocab].float().view(batch, rows, vocab)
    # How often each id stands in the sequence's text, and on the node's path in the tree.
    old = torch.arange(c["history"], device=DEV) < s["n"][:, None]
    times = torch.zeros(batch, vocab, device=DEV).scatter_add_(1, s["history"].long(), old.float())
    on_path = torch.zeros(batch, rows, vocab, device=DEV)
    on_path.scatter_add_(2, s["tokens"].long()[:, None, :].expand(batch, rows, rows), seen.float())
    times = times[:, None, :] + on_path
    repetition, frequency, presence = (p[:, None, None] for p in s["penalty"].unbind(1))
    x = torch.where(times > 0, torch.where(x > 0, x / repetition, x * repetition) - frequency * times - presence, x)
    # Each sequence's biases; of two for one id the last one counts.
    at = torch.arange(s["biases"], device=DEV)
    of = torch.searchsorted(s["bias_start"].long(), at, right=True) - 1
    last = torch.full((batch * vocab,), -1, device=DEV, dtype=torch.int64)
    last = last.scatter_reduce(0, of * vocab + s["bias_id"][:s["biases"]].long(), at, "amax")
    x = x + torch.where(last >= 0, s["bias"][last.clamp(min=0)], 0.0).view(batch, 1, vocab)
    x = x.view(batch * rows, vocab)
    if c["grammar"]:
        j = torch.arange(vocab, device=DEV)
        x = torch.where(((s["allow"][:, j // 32] >> (j % 32)) & 1) != 0, x, -math.inf)
    there = there.reshape(-1)
    out = torch.zeros_like(s["out"])
    out[:, :vocab] = torch.where(there[:, None], x, 0.0)  # rounded as it is stored; the pick is by the values before that
    best = x.amax(1, keepdim=True)
    first = torch.where(x == best, torch.arange(vocab, device=DEV, dtype=torch.int32), vocab).amin(1).int()
    some = best[:, 0] > -math.inf
    total = torch.exp(x - torch.where(some[:, None], best, 0.0)).sum(1)
    return (out, torch.where(there, torch.where(some, first, NONE), 0).int(),
            torch.where(there, torch.where(some, -torch.log(total), -math.inf), 0.0))


def _accept(s):
    c = s["case"]
    batch, rows, layers, d, cols = c["batch"], c["rows"], c["layers"], c["d"], c["cols"]
    if own:
        x, size = s["x"].data_ptr(), s["x"].element_size()
        _gpu().tree_accept(_tree(s), s["picks"].data_ptr(), x + size * d, x + size * 2 * d, 3 * d, batch * rows * 3 * d,
                           s["kv"].data_ptr(), cols * d, batch * cols * d, layers, cols, d, s["path"].data_ptr(),
                           s["kept"].data_ptr(), s["next"].data_ptr(), s["n_out"].data_ptr(), s["history"].data_ptr(), cols,
                           in16=c["half"])
        return {"kv": s["kv"].view(torch.float16), **{k: s[k] for k in ("path", "kept", "next", "n_out", "history")}}
    seen, there = _seen(s)
    i = torch.arange(rows, device=DEV)
    above = seen & (i[None, :] < i[:, None])
    parent = torch.where(above, i, -1).amax(2)
    agrees = (parent >= 0) & (s["tokens"] == s["picks"].gather(1, parent.clamp(min=0)))
    twin = (parent[:, :, None] == parent[:, None, :]) & agrees[:, None, :] & (i[None, :] < i[:, None])
    holds = (agrees & ~twin.any(2)) | (i == 0)
    on = there & (holds[:, None, :] | ~seen).all(2) & seen[:, :, 0]
    place = on.cumsum(1) - 1
    room = (cols - s["n"].clamp(0, cols))[:, None]
    on &= place < room
    kept = on.sum(1).int()
    b, node = on.nonzero(as_tuple=True)
    at = place[b, node]
    path = torch.full((batch, rows), -1, device=DEV, dtype=torch.int32)
    path[b, at] = node.int()
    last = path.gather(1, (kept[:, None] - 1).clamp(min=0).long()).clamp(min=0).long()
    after = torch.where(kept > 0, s["picks"].gather(1, last)[:, 0], s["tokens"][:, 0])
    n = s["n"].clamp(0, cols)
    history = s["history"].clone()
    history[b, n[b] + at] = s["tokens"][b, node]
    kv = s["kv"].view(torch.float16)
    k, v = s["x"][:, b, node, d:].half().view(layers, len(b), 2, d).unbind(2)
    where = (n[b] + at).long()
    kv[:, :, :cols * d].view(layers, batch, d // 2, cols, 2)[:, b, :, where, :] = k.view(layers, len(b), d // 2, 2).transpose(0, 1)
    kv[:, :, cols * d:].view(layers, batch, cols, d)[:, b, where] = v
    return {"kv": kv, "path": path, "kept": kept, "next": torch.where(s["count"] > 0, after, 0).int(), "n_out": n + kept, "history": history}


# --------------------------------------------------------------------------------------------- work


def work(case):
    batch, rows, size = case["batch"], case["rows"], 2 if case["half"] else 4
    nodes = batch * (rows + (rows + 1) // 2) / 2  # the nodes that are there, on average
    if case["kind"] == "attend":
        h, g, hd = case["heads"], case["kv_heads"], case["hd"]
        keys = (case["shortest"] + case["longest"]) / 2
        row = 2 * h * hd + (0 if case["cross"] else 2 * g * hd)
        pairs = nodes * (keys + (0 if case["cross"] else min(rows, 8)))
        return {"bytes": 4.0 * batch * keys * g * hd + size * nodes * row, "flops": 4.0 * pairs * h * hd}
    if case["kind"] == "rules":
        row = case["vocab"] * (2 * size + (1 / 8 if case["grammar"] else 0))
        return {"bytes": nodes * (row + 8) + batch * (3.0 * case["history"] + 6.0 * case["biases"]), "flops": 4.0 * nodes * case["vocab"]}
    moved = 2.0 * batch * case["kept"] * case["layers"] * case["d"]
    return {"bytes": moved * (size + 2) + 12.0 * batch * rows, "flops": 2.0 * moved}


# ----------------------------------------------------------------------------------- 64-bit passes


def _sees(mask, i, j):
    return (int(mask[i, j // 32]) >> (j % 32)) & 1


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "rules": _exact_rules, "accept": _exact_accept}[case["kind"]](s)


def _exact_attend(s):
    """Sequence by sequence and node by node's own list of keys, softmax(q.k / sqrt(hd)).v."""
    c = s["case"]
    h, g, hd, cols = c["heads"], c["kv_heads"], c["hd"], c["cols"]
    out = torch.zeros(c["batch"], c["rows"], h * hd, device=DEV, dtype=torch.float64)
    for b in range(c["batch"]):
        n, count = int(s["n"][b]), int(s["count"][b])
        mask = s["mask"][b].cpu().numpy()
        words = s["kv"][b].view(torch.float16).double()
        K = words[:cols * g * hd].reshape(g * hd // 2, cols, 2)[:, :n].permute(1, 0, 2).reshape(n, g, hd)
        V = words[cols * g * hd:].reshape(cols, g, hd)[:n]
        x = s["x"][b, :count]
        hidden = None
        if not c["cross"]:
            k, v = x[:, h * hd:].half().double().reshape(count, 2, g, hd).unbind(1)
            K, V = torch.cat([K, k]), torch.cat([V, v])
            hidden = torch.tensor([[not _sees(mask, i, j) for j in range(count)] for i in range(count)], device=DEV)
        if not len(K):
            continue
        q = x[:, :h * hd].double().reshape(count, h, hd)
        for head in range(h):
            of = head // (h // g)
            t = q[:, head] @ K[:, of].T / hd**0.5
            if hidden is not None:
                t[:, n:].masked_fill_(hidden, -math.inf)
            out[b, :count, head * hd:(head + 1) * hd] = torch.softmax(t, 1) @ V[:, of]
    return out


def _exact_rules(s):
    c = s["case"]
    vocab, rows = c["vocab"], c["rows"]
    out = torch.zeros(s["out"].shape, device=DEV, dtype=torch.float64)
    logprob = torch.zeros(len(out), device=DEV, dtype=torch.float64)
    start = s["bias_start"].tolist()
    for b in range(c["batch"]):
        text = s["history"][b, :int(s["n"][b])].long()
        mask = s["mask"][b].cpu().numpy()
        r, f, p = s["penalty"][b].double()
        bias = dict(zip(s["bias_id"][start[b]:start[b + 1]].tolist(), s["bias"][start[b]:start[b + 1]].tolist()))
        for i in range(int(s["count"][b])):
            path = torch.tensor([j for j in range(rows) if _sees(mask, i, j)], device=DEV)
            ids, times = torch.unique(torch.cat([text, s["tokens"][b, path].long()]), return_counts=True)
            x = s["logits"][b * rows + i, :vocab].double()
            t = x[ids]
            x[ids] = torch.where(t > 0, t / r, t * r) - f * times - p
            if bias:
                x[torch.tensor(list(bias), device=DEV)] += torch.tensor(list(bias.values()), device=DEV, dtype=torch.float64)
            if s["allow"] is not None:
                bits = s["allow"][b * rows + i].view(torch.uint8)
                x[((bits[:, None] >> torch.arange(8, device=DEV)) & 1).reshape(-1)[:vocab] == 0] = -math.inf
            out[b * rows + i, :vocab] = x
            best = x.max()
            logprob[b * rows + i] = -torch.logsumexp(x - best, 0) if best > -math.inf else -math.inf
    return out, None, logprob


def _exact_accept(s):
    """The caches after the step, from each sequence's walk down its tree; the whole numbers have no such value."""
    c = s["case"]
    d, cols = c["d"], c["cols"]
    kv = s["kv"].view(torch.float16).clone()
    for b in range(c["batch"]):
        n, count = int(s["n"][b]), int(s["count"][b])
        mask, tokens, picks = s["mask"][b].cpu().numpy(), s["tokens"][b].tolist(), s["picks"][b].tolist()
        at, node = n, 0 if count else None
        while node is not None and at < cols:
            k, v = s["x"][:, b, node, d:2 * d].half(), s["x"][:, b, node, 2 * d:].half()
            kv[:, b, :cols * d].view(-1, d // 2, cols, 2)[:, :, at] = k.reshape(-1, d // 2, 2)
            kv[:, b, cols * d:].view(-1, cols, d)[:, at] = v
            children = [i for i in range(node + 1, count) if max(j for j in range(i) if _sees(mask, i, j)) == node]
            at, node = at + 1, next((i for i in children if tokens[i] == picks[node]), None)
    return {"kv": kv.double(), "path": None, "kept": None, "next": None, "n_out": None, "history": None}
