"""Cases of the paged key/value cache: its page operations, the pass that norms, rotates and stores
the heads of new tokens, and attention for a batch whose sequences share a prefix.

The plain forms below say what each operator computes, in elementary torch operations.  With ``own``
set, ``run`` makes the calls a user makes of the framework.

Layouts.  k, v: [layers][pages][kv heads][page size][head dim] in f16 or bf16; table: int32
[sequences][pages of a row], -1 where a row holds no page; lens: int32 [sequences]; refs: int32
[pages], how many rows name the page.  Position p of sequence s lies in page table[s][p // page size].
"""

import importlib.util
import pathlib
import sys

import torch

own = False

ROOT = pathlib.Path(__file__).resolve().parent.parent
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _framework():
    name = "edgexpu_llm_b200"
    if name not in sys.modules:
        path = ROOT / "edgexpu-llm_b200"
        spec = importlib.util.spec_from_file_location(name, path / "__init__.py", submodule_search_locations=[str(path)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
        mod.init(0)
    from edgexpu_llm_b200 import kv

    return kv


# ---- cases -------------------------------------------------------------------------------------------
# Head layouts are those of the framework's two model shapes (9 query heads over 3 of 64, and 32 over 8
# of 128) and two generic ones (as many key as query heads; 96 wide).

LAYOUTS = [(9, 3, 64), (32, 8, 128), (32, 8, 128), (20, 20, 64), (12, 2, 96)]


def listed():
    return [
        # one new token of one request, small model, no head norm: the shortest pass there is
        {"name": "heads_one_token", "op": "heads", "batch": 1, "each": 1, "heads": 9, "kv": 3, "dim": 64, "type": "f16",
         "norm": False, "pairing": "adjacent", "rot": 64, "page": 16, "pads": 0, "fused": False, "start": 511},
        # a decode step of 61 requests in a batch padded to 64, heads normed, q|k|v in one buffer
        {"name": "heads_decode_64", "op": "heads", "batch": 61, "each": 1, "heads": 32, "kv": 8, "dim": 128, "type": "bf16",
         "norm": True, "pairing": "halves", "rot": 128, "page": 64, "pads": 3, "fused": True, "start": 9000},
        # four prompts of 2047 tokens read in one pass
        {"name": "heads_prompt_8k", "op": "heads", "batch": 4, "each": 2047, "heads": 32, "kv": 8, "dim": 128, "type": "f16",
         "norm": True, "pairing": "adjacent", "rot": 128, "page": 64, "pads": 4, "fused": False, "start": 0},
        # a single request's decode step: nothing shared, a short cache
        {"name": "attend_one_short", "op": "attend", "batch": 1, "queries": 1, "shared": 0, "own_min": 117, "own_max": 117,
         "heads": 9, "kv": 3, "dim": 64, "type": "f16", "page": 16, "idle": 0},
        # a decode step of 32 requests (two slots of the batch idle) behind one 4k prompt
        {"name": "attend_decode_32", "op": "attend", "batch": 32, "queries": 1, "shared": 4001, "own_min": 1, "own_max": 511,
         "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "page": 64, "idle": 2},
        # the largest decode step: 128 requests behind a 32k prompt
        {"name": "attend_decode_128", "op": "attend", "batch": 128, "queries": 1, "shared": 32768, "own_min": 33,
         "own_max": 2000, "heads": 32, "kv": 8, "dim": 128, "type": "f16", "page": 64, "idle": 0},
        # 32 users' questions of 1 to 64 tokens read in one pass behind an 8k prompt, small pages
        {"name": "attend_questions", "op": "attend", "batch": 32, "queries": 64, "shared": 8190, "own_min": 64, "own_max": 200,
         "heads": 32, "kv": 8, "dim": 128, "type": "f16", "page": 16, "idle": 0},
        # a speculative step: rejected tokens' pages go back and room for the next guesses is taken
        {"name": "pages_step_64", "op": "step", "batch": 64, "len_min": 100, "len_max": 4000, "drop": 5, "new": 6,
         "layers": 2, "kv": 8, "dim": 128, "type": "f16", "page": 16, "spare": 100},
        # 128 requests start from one prompt: the old ones go, the prompt is forked, its last page copied
        {"name": "pages_fork_128", "op": "fork", "batch": 128, "prompt": 8191, "new": 40, "layers": 16, "kv": 8, "dim": 128,
         "type": "bf16", "page": 64, "spare": 64},
        # a fragmented pool is packed to its lower end
        {"name": "pages_compact", "op": "compact", "batch": 48, "len_min": 1, "len_max": 4000, "layers": 16, "kv": 8,
         "dim": 128, "type": "f16", "page": 64, "spare": 500},
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def _drawn(rng):
    op = rng.choice(["heads", "attend", "attend", "step", "fork", "compact", "copy"])
    heads, kv, dim = rng.choice(LAYOUTS)
    c = {"op": op, "kv": kv, "dim": dim, "type": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 32, 64, 128])}
    if op == "heads":
        each = rng.choice([1, 1, _log(rng, 2, 2047)])
        return c | {"batch": _log(rng, 1, 128) if each == 1 else _log(rng, 1, 8), "each": each, "heads": heads,
                    "norm": rng.random() < 0.7, "pairing": rng.choice(["adjacent", "halves"]),
                    "rot": rng.choice([dim, dim, dim // 2]), "pads": rng.choice([0, 0, 3]), "fused": rng.random() < 0.5,
                    "start": _log(rng, 1, 16000) - 1}
    if op == "attend":
        queries = rng.choice([1, 1, 1, _log(rng, 2, 64)])
        own_min = _log(rng, max(1, queries), 1000)
        batch = _log(rng, 1, 128) if queries == 1 else _log(rng, 1, 32)
        return c | {"batch": batch, "queries": queries, "shared": rng.choice([0, _log(rng, 1, 32768), _log(rng, 1, 32768)]),
                    "own_min": own_min, "own_max": _log(rng, own_min, 2000), "heads": heads,
                    "idle": rng.choice([0, 0, min(2, batch - 1)])}
    if op == "step":
        len_min = _log(rng, 20, 1000)
        return c | {"batch": _log(rng, 1, 128), "len_min": len_min, "len_max": _log(rng, len_min, 4000),
                    "drop": rng.randint(0, 20), "new": rng.randint(1, 100), "layers": rng.randint(1, 2),
                    "spare": _log(rng, 1, 2000)}
    if op == "fork":
        return c | {"batch": _log(rng, 1, 128), "prompt": _log(rng, 1, 8191), "new": _log(rng, 1, 100),
                    "layers": _log(rng, 1, 16), "spare": _log(rng, 1, 500)}
    if op == "compact":
        len_min = _log(rng, 1, 500)
        return c | {"batch": _log(rng, 1, 48), "len_min": len_min, "len_max": _log(rng, len_min, 4000),
                    "layers": _log(rng, 1, 16), "spare": _log(rng, 10, 500)}
    return c | {"moves": _log(rng, 1, 200), "layers": _log(rng, 1, 16), "spare": _log(rng, 10, 500)}


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["op"], {"bytes": 0, "flops": 0})
        most[c["op"]] = {k: max(m[k], w[k]) for k in m}
    most["copy"] = most["fork"]
    while True:
        c = _drawn(rng)
        w, top = work(c), most[c["op"]]
        if w["bytes"] <= top["bytes"] and w["flops"] <= max(top["flops"], 0):
            return c


def _spread(lo, hi, n):
    """n lengths from lo to hi, neither sorted nor equal."""
    return [lo + (i * 7919 + 13) % (hi - lo + 1) for i in range(n)]


def _lens(c):
    """Of each entry of an attend case: its sequence's length and its new tokens (0 for an idle slot)."""
    n_q = [1 + (i * 37 + 5) % c["queries"] for i in range(c["batch"])]
    own_len = _spread(max(c["own_min"], c["queries"]), max(c["own_max"], c["queries"]), c["batch"])
    idle = c["batch"] - c["idle"]
    return [c["shared"] + o for o in own_len], [q if i < idle else 0 for i, q in enumerate(n_q)]


def _up(a, b):
    return -(-a // b)


def work(c):
    row = c["kv"] * c["dim"] * 2 * 2  # K and V of one token in one layer
    if c["op"] == "heads":
        n, width = c["batch"] * c["each"], (c["heads"] + 2 * c["kv"]) * c["dim"]
        return {"bytes": n * (width * 6 + 4 * c["rot"] + 8) + c["pads"] * (2 * c["heads"] * c["dim"]),
                "flops": n * width * (6 if c["norm"] else 3)}
    if c["op"] == "attend":
        lens, n_q = _lens(c)
        live = [(ln, q) for ln, q in zip(lens, n_q) if q]
        vis = sum(q * (ln - q) + q * (q + 1) // 2 for ln, q in live)
        held = c["shared"] + sum(ln - c["shared"] for ln, _ in live)
        return {"bytes": held * row + sum(q for _, q in live) * c["heads"] * c["dim"] * 4,
                "flops": 4 * c["dim"] * c["heads"] * vis}
    if c["op"] == "step":
        return {"bytes": 8 * (c["batch"] * 4 + _pool(c)[0]) + c["batch"] * 16, "flops": 0}
    if c["op"] == "fork":
        tail, pages = c["prompt"] % c["page"], _up(c["prompt"], c["page"])
        return {"bytes": c["batch"] * (2 * tail * row * c["layers"] + 8 * pages) + 8 * _pool(c)[0], "flops": 0}
    if c["op"] == "copy":
        return {"bytes": 2 * c["moves"] * c["page"] * row * c["layers"], "flops": 0}
    moved = sum(1 for p in _scattered(c) if p >= _live(c))
    return {"bytes": 2 * moved * c["page"] * row * c["layers"] + 8 * (_pool(c)[0] + _live(c)), "flops": 0}


# ---- what a user has in hand -------------------------------------------------------------------------


def _held(c):
    """Pages of each sequence at the start of a page case."""
    if c["op"] == "fork":
        return [_up(c["prompt"], c["page"])] + [0] * c["batch"]
    if c["op"] == "copy":
        return []
    return [_up(n, c["page"]) for n in _spread(c["len_min"], c["len_max"], c["batch"])]


def _live(c):
    return sum(_held(c))


def _pool(c):
    """Pages of the pool, and of a table row."""
    held = _held(c)
    if c["op"] == "copy":
        return 2 * c["moves"] + c["spare"], 1
    if c["op"] == "fork":
        return held[0] + c["batch"] * (_up(c["new"], c["page"]) + 1) + c["spare"], held[0] + _up(c["new"], c["page"]) + 1
    extra = _up(c.get("new", 0), c["page"]) + 1
    return sum(held) + c["batch"] * extra + c["spare"], max(held) + extra


def _scattered(c):
    """The pages of the sequences of a page case, in an order that leaves holes all over the pool."""
    n = _pool(c)[0]
    step = next(s for s in range(max(1, int(n * 0.618)), 2 * n + 2) if _gcd(s, n) == 1)
    return [(i * step + 3) % n for i in range(_live(c))]


def _gcd(a, b):
    while b:
        a, b = b, a % b
    return a


def _normal(shape, seed, dtype):
    """Standard normal values, drawn in the type itself where the pool is large."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache(c, layers, pages, seed, table, lens):
    """Pools full of numbers and the tables over them."""
    shape = (layers, pages, c["kv"], c["page"], c["dim"])
    s = {"k": _normal(shape, seed * 4 + 1, DTYPES[c["type"]]), "v": _normal(shape, seed * 4 + 2, DTYPES[c["type"]])}
    s["table"], s["lens"] = table, _ints(lens)
    named = table[table >= 0].long()
    s["refs"] = torch.zeros(pages, dtype=torch.int32, device="cuda").index_add_(0, named, torch.ones_like(named, dtype=torch.int32))
    if own:
        s["cache"] = _framework().KvCache(s["k"], s["v"], s["table"], s["lens"], s["refs"])
    return s


def _rope_table(positions, rot):
    """cos and sin of every pair, [positions][rot]: the layout of the framework's decoder."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).reshape(positions, rot).float()


def _rows(counts, pages, columns, seed):
    """A table whose row i holds counts[i] pages of its own, in random order."""
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=gen, dtype=torch.int64).tolist()
    table, at = [[-1] * columns for _ in counts], 0
    for row, n in zip(table, counts):
        row[:n] = order[at:at + n]
        at += n
    return table


def prepare(c, seed):
    if c["op"] == "heads":
        return _prepare_heads(c, seed)
    if c["op"] == "attend":
        return _prepare_attend(c, seed)
    pages, columns = _pool(c)
    held = _held(c)
    where = _scattered(c) if c["op"] != "copy" else []
    table, at = [[-1] * columns for _ in held] or [[-1]], 0
    for row, n in zip(table, held):
        row[:n] = where[at:at + n]
        at += n
    lens = ([c["prompt"]] + [0] * c["batch"] if c["op"] == "fork" else [0] if c["op"] == "copy"
            else _spread(c["len_min"], c["len_max"], c["batch"]))
    s = _cache(c, c["layers"], pages, seed, _ints(table), lens) | {"op": c["op"]}
    if c["op"] == "copy":
        gen = torch.Generator().manual_seed(seed)
        order = torch.randperm(pages, generator=gen)[: 2 * c["moves"]].to(torch.int32).cuda()
        return s | {"src": order[: c["moves"]].contiguous(), "dst": order[c["moves"]:].contiguous()}
    if c["op"] == "fork":
        return s | {"src": _ints([0] * c["batch"]), "dst": _ints(list(range(1, c["batch"] + 1))),
                    "new": _ints([1 + (i * 31 + seed) % c["new"] for i in range(c["batch"])])}
    if c["op"] == "step":
        gen = torch.Generator().manual_seed(seed)
        drop = torch.randint(0, c["drop"] + 1, (c["batch"],), generator=gen, dtype=torch.int32).cuda()
        return s | {"seqs": torch.randperm(c["batch"], generator=gen).to(torch.int32).cuda(),
                    "keep": (s["lens"] - drop).clamp(min=0), "new": _ints([c["new"]] * c["batch"])}
    # the scheduler's own copy of the tables, from before the last packing
    return s | {"was": (s["table"].clone(), s["refs"].clone())}


def _prepare_heads(c, seed):
    batch, each, total = c["batch"], c["each"], c["batch"] * c["each"]
    ends = [c["start"] + each + (i * 7 % 5) for i in range(batch)]
    held = [_up(e, c["page"]) for e in ends]
    pages = sum(held) + 3
    s = _cache(c, 1, pages, seed, _ints(_rows(held, pages, max(held), seed)), ends)
    widths = [c["heads"] * c["dim"], c["kv"] * c["dim"], c["kv"] * c["dim"]]
    n = total + c["pads"]
    if c["fused"]:
        q, k, v = _normal((n, sum(widths)), seed * 4 + 3, torch.float32).split(widths, 1)
    else:
        q, k, v = (_normal((n, w), seed * 4 + 3 + 1000 * i, torch.float32) for i, w in enumerate(widths))
    weights = 1 + 0.1 * _normal((2, c["dim"]), seed * 4 + 7, torch.float32)
    seqs = [i for i in range(batch) for _ in range(each)] + [-1] * c["pads"]
    pos = [ends[i] - each + j for i in range(batch) for j in range(each)] + [0] * c["pads"]
    return s | {"op": "heads", "q": q, "knew": k, "vnew": v, "qw": weights[0] if c["norm"] else None,
                "kw": weights[1] if c["norm"] else None, "rope": _rope_table(max(ends), c["rot"]), "seqs": _ints(seqs),
                "pos": _ints(pos), "heads": c["heads"], "pairing": c["pairing"], "eps": 1e-5}


def _prepare_attend(c, seed):
    by_entry, n_q = _lens(c)
    ps, shared, batch = c["page"], c["shared"], c["batch"]
    order = [1 + (i * 5 + 2) % batch if batch % 5 else 1 + i for i in range(batch)]  # the rows of the batch's entries
    lens = [n for _, n in sorted(zip(order, by_entry))]
    full = shared // ps  # pages that all rows name; a page that the prefix fills in part is each row's own copy
    own_pages = [_up(n, ps) - full for n in lens]
    prompt_pages = _up(shared, ps)
    pages = prompt_pages + sum(own_pages) + 2
    rows = _rows([prompt_pages] + own_pages, pages, prompt_pages + max(own_pages), seed)
    table = [rows[0]] + [(rows[0][:full] + r)[: len(r)] for r in rows[1:]]
    s = _cache(c, 1, pages, seed, _ints(table), [shared] + lens)
    table_t = s["table"].long()
    if shared % ps:  # the copies of the prompt's last page
        for pool in (s["k"], s["v"]):
            pool[0, table_t[1:, full], :, : shared % ps] = pool[0, table_t[0, full], :, : shared % ps]
    for i, n in enumerate([shared] + lens):  # memory past a sequence's end holds anything
        if n % ps:
            s["k"][0, table_t[i, n // ps], :, n % ps:] = float("nan")
            s["v"][0, table_t[i, n // ps], :, n % ps:] = float("nan")
    starts = [0]
    for q in n_q:
        starts.append(starts[-1] + q if c["queries"] > 1 else starts[-1] + 1)
    rows_of = [order[i] if n_q[i] else -1 for i in range(batch)]
    # every entry's new tokens are the last of its sequence
    q = _normal((starts[-1], c["heads"], c["dim"]), seed * 4 + 3, DTYPES[c["type"]])
    return s | {"op": "attend", "q": q, "seqs": _ints(rows_of), "q_start": _ints(starts) if c["queries"] > 1 else None,
                "shared": shared, "queries": c["queries"], "max_len": max(lens), "own_max": max(lens) - shared,
                "scale": c["dim"] ** -0.5, "entry": _ints([i for i in range(batch) for _ in range(starts[i + 1] - starts[i])]).long(),
                "at": _ints([j for i in range(batch) for j in range(starts[i + 1] - starts[i])]).long(),
                "starts": _ints(starts).long()}


# ---- one pass ----------------------------------------------------------------------------------------


def run(s):
    op = s["op"]
    if op == "heads":
        q = _own_heads(s) if own else _heads(s)
        return {"q": q, "k": s["k"], "v": s["v"]}
    if op == "attend":
        return {"out": _own_attend(s) if own else _attend(s)}
    pages = s["cache"] if own else s
    free, fork, append, copy, compact = _OWN_PAGES if own else _PLAIN_PAGES
    if op == "copy":
        copy(pages, s["src"], s["dst"])
        return {"k": s["k"], "v": s["v"]}
    if op == "fork":
        free(pages, s["dst"], None)
        fork(pages, s["src"], s["dst"])
        extra = append(pages, s["dst"], s["new"])
    elif op == "step":
        free(pages, s["seqs"], s["keep"])
        extra = append(pages, s["seqs"], s["new"])
    else:
        s["table"].copy_(s["was"][0])
        s["refs"].copy_(s["was"][1])
        extra = compact(pages)
    return {"table": s["table"], "refs": s["refs"], "lens": s["lens"], "extra": extra, "k": s["k"], "v": s["v"]}


def _own_heads(s):
    return s["cache"].qk_norm_rope(0, s["q"], s["knew"], s["vnew"], s["seqs"], s["pos"], n_heads=s["heads"], q_norm=s["qw"],
                                   k_norm=s["kw"], eps=s["eps"], rope=s["rope"], pairing=s["pairing"])


def _own_attend(s):
    return s["cache"].attention(0, s["q"], s["seqs"], q_start=s["q_start"], shared_seq=0, shared_len=s["shared"],
                                max_len=s["max_len"], scale=s["scale"])


_OWN_PAGES = (lambda c, seqs, keep: c.free(seqs, keep), lambda c, src, dst: c.fork(src, dst),
              lambda c, seqs, new: c.append(seqs, new), lambda c, src, dst: c.copy(src, dst), lambda c: c.compact())


# ---- plain forms -------------------------------------------------------------------------------------


def _norm_rotate(x, w, eps, angles, halves):
    """x: [tokens][heads][dim] fp32; angles: [tokens][rot] cos and sin of each pair."""
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    rot = angles.shape[-1]
    cos, sin = angles[:, None, 0::2], angles[:, None, 1::2]
    turned, rest = x[..., :rot], x[..., rot:]
    a, b = (turned[..., : rot // 2], turned[..., rot // 2:]) if halves else (turned[..., 0::2], turned[..., 1::2])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _heads(s):
    layers, pages, kv, ps, dim = s["k"].shape
    n, dtype, halves = s["q"].shape[0], s["k"].dtype, s["pairing"] == "halves"
    live = s["seqs"] >= 0
    angles = s["rope"][s["pos"].long()]
    q = _norm_rotate(s["q"].reshape(n, s["heads"], dim), s["qw"], s["eps"], angles, halves)
    k = _norm_rotate(s["knew"].reshape(n, kv, dim), s["kw"], s["eps"], angles, halves).to(dtype)
    v = s["vnew"].reshape(n, kv, dim).to(dtype)
    page = s["table"][s["seqs"].long().clamp(min=0), (s["pos"] // ps).long()].long()
    # padding tokens write the first token's values once more
    at = torch.where(live, torch.arange(n, device=q.device), 0)
    page, off = page[at], (s["pos"] % ps).long()[at]
    s["k"][0, page, :, off] = k[at]
    s["v"][0, page, :, off] = v[at]
    return torch.where(live[:, None, None], q, 0.0).to(dtype)


def _attend(s):
    kp, vp, q, table, lens = s["k"][0], s["v"][0], s["q"], s["table"].long(), s["lens"].long()
    pages, kv, ps, dim = kp.shape
    seqs, batch, nq, shared = s["seqs"].long(), s["seqs"].shape[0], s["queries"], s["shared"]
    rows, live, dev = table[seqs.clamp(min=0)], seqs >= 0, q.device
    count = s["starts"][1:] - s["starts"][:-1]
    j = torch.arange(nq, device=dev)
    pick = (s["starts"][:-1, None] + j).clamp(max=q.shape[0] - 1)
    qq = q[pick].float().reshape(batch, nq, kv, -1, dim) * s["scale"]
    visible = torch.where(live[:, None] & (j < count[:, None]), lens[seqs.clamp(min=0), None] - count[:, None] + j + 1, 0)
    # the prefix, once for the whole batch
    n_pre = _up(shared, ps)
    kpre = kp[table[0, :n_pre]].transpose(0, 1).reshape(kv, n_pre * ps, dim)[:, :shared].float()
    vpre = vp[table[0, :n_pre]].transpose(0, 1).reshape(kv, n_pre * ps, dim)[:, :shared].float()
    s_pre = torch.einsum("bqhgd,hpd->bqhgp", qq, kpre)
    at = torch.arange(shared, device=dev)
    s_pre = s_pre.masked_fill_((at >= visible[:, :, None])[:, :, None, None], float("-inf"))
    # each sequence's own positions
    at = shared + torch.arange(s["own_max"], device=dev)
    column = (at // ps).clamp(max=table.shape[1] - 1)
    page, off = rows[:, column].clamp(min=0), (at % ps).expand(batch, -1)
    held = live[:, None] & (at < lens[seqs.clamp(min=0), None])
    kown = torch.where(held[:, :, None, None], kp[page, :, off].float(), 0.0)
    vown = torch.where(held[:, :, None, None], vp[page, :, off].float(), 0.0)
    s_own = torch.einsum("bqhgd,bshd->bqhgs", qq, kown)
    s_own = s_own.masked_fill_((at >= visible[:, :, None])[:, :, None, None], float("-inf"))
    top = s_own.amax(-1, keepdim=True)
    if shared:
        top = torch.maximum(top, s_pre.amax(-1, keepdim=True))
    top = torch.where(torch.isinf(top), 0.0, top)
    p_pre, p_own = (s_pre - top).exp(), (s_own - top).exp()
    total = p_pre.sum(-1, keepdim=True) + p_own.sum(-1, keepdim=True)
    out = torch.einsum("bqhgp,hpd->bqhgd", p_pre, vpre) + torch.einsum("bqhgs,bshd->bqhgd", p_own, vown)
    out = torch.where(total > 0, out / total, 0.0).reshape(batch, nq, -1, dim)
    return out[s["entry"], s["at"]].to(q.dtype)


def _free(s, seqs, keep):
    seqs, ps = seqs.long(), s["k"].shape[3]
    keep = torch.zeros_like(seqs, dtype=torch.int32) if keep is None else keep
    kept = torch.minimum(s["lens"][seqs], keep)
    rows = s["table"][seqs]
    gone = (torch.arange(rows.shape[1], device=rows.device) >= ((kept + ps - 1) // ps)[:, None]) & (rows >= 0)
    s["refs"].index_add_(0, rows.clamp(min=0).flatten().long(), -gone.int().flatten())
    s["table"][seqs] = torch.where(gone, -1, rows)
    s["lens"][seqs] = kept


def _fork(s, src, dst):
    src, dst = src.long(), dst.long()
    rows = s["table"][src]
    s["table"][dst] = rows
    s["lens"][dst] = s["lens"][src]
    s["refs"].index_add_(0, rows.clamp(min=0).flatten().long(), (rows >= 0).int().flatten())


def _append(s, seqs, new):
    """Pages for new[i] more tokens of each sequence; the position of the first of them."""
    seqs, ps, dev = seqs.long(), s["k"].shape[3], seqs.device
    held, rows = s["lens"][seqs], s["table"][seqs]
    first, last = (held + ps - 1) // ps, (held + new + ps - 1) // ps
    # a last page that another row names too is copied; the batch's later rows see one sharer fewer
    old = rows.gather(1, (held // ps).long().clamp(max=rows.shape[1] - 1)[:, None])[:, 0]
    part = (held % ps > 0) & (new > 0)
    alike = (old[:, None] == old) & part[:, None] & part
    earlier = torch.tril(alike, -1).sum(1)
    split = part & (s["refs"][old.clamp(min=0).long()] - earlier > 1)
    first = first - split.int()
    need = last - first
    offset = need.cumsum(0) - need
    unused = torch.argsort((s["refs"] > 0).int(), stable=True)  # free pages first, lowest first
    fits = need.sum() <= (s["refs"] <= 0).sum()
    column = torch.arange(rows.shape[1], device=dev)
    fresh = (column >= first[:, None]) & (column < last[:, None]) & fits
    rank = (offset[:, None] + column - first[:, None]).clamp(min=0, max=unused.shape[0] - 1)
    page = unused[rank].int()
    s["table"][seqs] = torch.where(fresh, page, rows)
    one = torch.ones_like(page).flatten()
    s["refs"].index_add_(0, page.flatten().long(), (one * fresh.flatten()).int())
    split = split & fits
    s["refs"].index_add_(0, old.clamp(min=0).long(), -split.int())
    into = torch.where(split, page.gather(1, first.long().clamp(max=rows.shape[1] - 1)[:, None])[:, 0], -1)
    done = torch.nonzero(split)[:, 0]
    if done.numel():
        a, b, token = old[done].long(), into[done].long(), torch.arange(ps, device=dev)
        valid = (token < (held % ps)[done, None])[None, :, None, :, None]
        for pool in (s["k"], s["v"]):
            pool[:, b] = torch.where(valid, pool[:, a], pool[:, b])
    s["lens"][seqs] = torch.where(fits, held + new, held)
    return torch.where(fits, held, -1)


def _copy(s, src, dst):
    for pool in (s["k"], s["v"]):
        pool[:, dst.long()] = pool[:, src.long()]


def _compact(s):
    live = s["refs"] > 0
    n = live.sum()
    index = torch.arange(live.shape[0], device=live.device)
    src, dst = torch.nonzero(live & (index >= n))[:, 0], torch.nonzero(~live & (index < n))[:, 0]
    _copy(s, src, dst)
    to = index.clone()
    to[src] = dst
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()].int(), -1))
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    return n.int()


_PLAIN_PAGES = (_free, _fork, _append, _copy, _compact)


# ---- the definitions in 64 bits ----------------------------------------------------------------------


def exact(c, seed):
    if c["op"] == "heads":
        return _exact_heads(prepare(c, seed))
    if c["op"] == "attend":
        return _exact_attend(prepare(c, seed))
    return None  # moves whole numbers and copies


def _exact_heads(s):
    dim, ps = s["k"].shape[-1], s["k"].shape[3]
    n, kv = s["q"].shape[0], s["k"].shape[2]
    turn = torch.zeros(n, dim // 2, dtype=torch.complex128, device="cuda") + 1
    rot = s["rope"].shape[1]
    angle = s["rope"].double()[s["pos"].long()]
    turn[:, : rot // 2] = torch.complex(angle[:, 0::2], angle[:, 1::2])

    def heads(x, w, count):
        x = x.double().reshape(n, count, dim)
        if w is not None:
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / dim + s["eps"]) * w.double()
        if s["pairing"] == "halves":  # pair j of the turned part is (j, j + rot / 2)
            order = torch.cat([torch.stack([torch.arange(rot // 2), torch.arange(rot // 2) + rot // 2], 1).flatten(), torch.arange(rot, dim)])
        else:
            order = torch.arange(dim)
        order = order.to(x.device)
        z = torch.view_as_complex(x[..., order].reshape(n, count, dim // 2, 2).contiguous()) * turn[:, None]
        y = torch.empty_like(x)
        y[..., order] = torch.view_as_real(z).reshape(n, count, dim)
        return y

    q, k = heads(s["q"], s["qw"], s["heads"]), heads(s["knew"], s["kw"], kv)
    kp, vp = s["k"].double(), s["v"].double()
    t = torch.nonzero(s["seqs"] >= 0)[:, 0]
    page, off = s["table"][s["seqs"][t].long(), (s["pos"][t] // ps).long()].long(), (s["pos"][t] % ps).long()
    kp[0, page, :, off] = k[t]
    vp[0, page, :, off] = s["vnew"].double().reshape(n, kv, dim)[t]
    q[s["seqs"] < 0] = 0
    return {"q": q, "k": kp, "v": vp}


def _exact_attend(s):
    kv, ps, dim = s["k"].shape[2:]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, seqs, lens = s["starts"].tolist(), s["seqs"].tolist(), s["lens"].tolist()
    for i, row in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        if row < 0 or a == b:
            continue
        n = lens[row]
        pages = s["table"][row, : _up(n, ps)].long()
        k = s["k"][0, pages].double().transpose(1, 2).reshape(-1, kv, dim)[:n]
        v = s["v"][0, pages].double().transpose(1, 2).reshape(-1, kv, dim)[:n]
        q = s["q"][a:b].double().reshape(b - a, kv, -1, dim)
        for h in range(kv):
            for at in range(0, b - a, 16):
                qq = q[at:at + 16, h]
                score = (qq @ k[:, h].T) * s["scale"]
                seen = n - (b - a) + at + torch.arange(qq.shape[0], device="cuda") + 1
                score = score.masked_fill(torch.arange(n, device="cuda") >= seen[:, None, None], float("-inf"))
                out[a + at:a + at + qq.shape[0]].view(qq.shape[0], kv, -1, dim)[:, h] = torch.softmax(score, -1) @ v[:, h]
    return {"out": out}
