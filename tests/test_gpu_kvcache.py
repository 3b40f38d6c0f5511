"""The paged cache: its page operations against a plain model of the state, and the pass that norms,
rotates and stores new heads against the formulas in 64 bits."""

import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def kv(gpu):
    from edgexpu_llm_b200 import kv as module

    return module


def sync_error(gpu):
    """The message of the next stream sync ("" if it succeeds)."""
    buf = ctypes.create_string_buffer(512)
    ok = gpu.load_cuda().edgexpu_cuda_stream_sync(torch.cuda.current_stream().cuda_stream, buf, 512)
    return "" if ok else buf.value.decode()


def ints(*v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


class Model:
    """The state of a cache in plain lists, one operation after the other."""

    def __init__(self, cache):
        self.ps = cache.k.shape[3]
        self.k, self.v = cache.k.cpu().clone(), cache.v.cpu().clone()
        self.n_pages, (self.n_seqs, self.columns) = cache.k.shape[1], cache.table.shape
        self.rows = [[] for _ in range(self.n_seqs)]
        self.lens = [0] * self.n_seqs
        self.refs = [0] * self.n_pages

    def up(self, n):
        return -(-n // self.ps)

    def append(self, seqs, new):
        free = [p for p in range(self.n_pages) if self.refs[p] == 0]
        refs, plan, taken = list(self.refs), [], 0
        for s, n in zip(seqs, new):
            held = self.lens[s]
            split = n > 0 and held % self.ps != 0 and refs[self.rows[s][-1]] > 1
            if split:
                refs[self.rows[s][-1]] -= 1
            count = self.up(held + n) - self.up(held) + split
            plan.append((s, n, split, count))
            taken += count
        if taken > len(free):
            return [-1] * len(seqs), taken - len(free)
        pos = []
        for s, n, split, count in plan:
            pages, free = free[:count], free[count:]
            pos.append(self.lens[s])
            if split:
                old, tail = self.rows[s].pop(), self.lens[s] % self.ps
                self.refs[old] -= 1
                for pool in (self.k, self.v):
                    pool[:, pages[0], :, :tail] = pool[:, old, :, :tail]
            self.rows[s] += pages
            for p in pages:
                self.refs[p] = 1
            self.lens[s] += n
        return pos, 0

    def fork(self, src, dst):
        for s, d in zip(src, dst):
            self.rows[d], self.lens[d] = list(self.rows[s]), self.lens[s]
            for p in self.rows[s]:
                self.refs[p] += 1

    def free(self, seqs, keep):
        for s, n in zip(seqs, keep):
            n = min(n, self.lens[s])
            for p in self.rows[s][self.up(n):]:
                self.refs[p] -= 1
            self.rows[s], self.lens[s] = self.rows[s][: self.up(n)], n

    def copy(self, src, dst):
        for pool in (self.k, self.v):
            pool[:, dst] = pool[:, src].clone()

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        src = [p for p in range(live, self.n_pages) if self.refs[p] > 0]
        dst = [p for p in range(live) if self.refs[p] == 0]
        to = dict(zip(src, dst))
        if src:
            self.copy(src, dst)
        for s, d in to.items():
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]
        return live

    def check(self, cache):
        table = torch.full((self.n_seqs, self.columns), -1, dtype=torch.int32)
        for i, row in enumerate(self.rows):
            table[i, : len(row)] = torch.tensor(row, dtype=torch.int32)
        assert cache.lens.tolist() == self.lens
        assert cache.refs.tolist() == self.refs
        assert torch.equal(cache.table.cpu(), table)
        assert torch.equal(cache.k.cpu().view(torch.int16), self.k.view(torch.int16))
        assert torch.equal(cache.v.cpu().view(torch.int16), self.v.view(torch.int16))


def filled(kv, layers, pages, ps, n_kv, dim, n_seqs, columns, dtype=torch.float16, interleaved=False):
    """An empty cache whose pools hold numbers."""
    if interleaved:  # k and v of a page side by side, one row of pages spare: page and layer strides of their own
        pool = torch.randn(layers, pages + 1, 2, n_kv, ps, dim, device="cuda").to(dtype)
        k, v = pool[:, :pages, 0], pool[:, :pages, 1]
    else:
        k, v = (torch.randn(layers, pages, n_kv, ps, dim, device="cuda").to(dtype) for _ in range(2))
    return kv.KvCache(k, v, torch.full((n_seqs, columns), -1, dtype=torch.int32, device="cuda"),
                      torch.zeros(n_seqs, dtype=torch.int32, device="cuda"), torch.zeros(pages, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("ps,layers,n_kv,dim,pages,interleaved", [
    (16, 1, 1, 8, 40, False), (16, 3, 2, 64, 300, True), (64, 2, 3, 128, 90, False), (256, 1, 2, 72, 33, True),
    (32, 2, 1, 256, 5000, False)])
def test_random_operations_match_the_model(gpu, kv, ps, layers, n_kv, dim, pages, interleaved):
    torch.manual_seed(ps + dim)
    rng = np.random.default_rng(ps * dim)
    n_seqs, columns = 23, 9
    cache = filled(kv, layers, pages, ps, n_kv, dim, n_seqs, columns, interleaved=interleaved)
    model = Model(cache)
    missing = ints(77)
    for step in range(60):
        op = rng.choice(["append", "append", "append", "fork", "fork", "free", "free", "compact", "copy"])
        if op == "append":
            seqs = rng.permutation(n_seqs)[: rng.integers(1, n_seqs + 1)].tolist()
            new = [int(min(rng.choice([0, 1, ps // 2 + 1, 3 * ps]), columns * ps - model.lens[s])) for s in seqs]
            pos = cache.append(ints(*seqs), ints(*new), missing=missing)
            want, short = model.append(seqs, new)
            assert pos.tolist() == want and missing.item() == short
        elif op == "fork":
            empty = [s for s in range(n_seqs) if model.lens[s] == 0]
            dst = rng.permutation(empty).tolist()[: rng.integers(0, len(empty) + 1)]
            src = [int(s) for s in rng.choice([s for s in range(n_seqs) if s not in dst], len(dst))] if len(dst) < n_seqs else []
            dst = dst[: len(src)]
            cache.fork(ints(*src), ints(*dst))
            model.fork(src, dst)
        elif op == "free":
            seqs = rng.permutation(n_seqs)[: rng.integers(1, n_seqs)].tolist()
            keep = [int(rng.choice([0, 0, model.lens[s], model.lens[s] // 2, model.lens[s] + 5])) for s in seqs]
            cache.free(ints(*seqs), ints(*keep))
            model.free(seqs, keep)
        elif op == "compact":
            assert cache.compact().item() == model.compact()
        else:
            order = rng.permutation(pages)
            n = int(rng.integers(0, min(pages // 2, 20)))
            src, dst = order[:n].tolist(), order[n:2 * n].tolist()
            cache.copy(ints(*src), ints(*dst))
            model.copy(src, dst)
        model.check(cache)
    assert sync_error(gpu) == ""


def test_a_shared_last_page_is_copied_for_all_but_its_last_holder(kv):
    cache = filled(kv, 2, 64, 16, 2, 64, 8, 4)
    model = Model(cache)
    for op, args in [("append", ([0], [21])), ("fork", ([0, 0, 0], [3, 1, 2])), ("append", ([2, 0, 3], [1, 40, 0])),
                     ("append", ([3, 1], [2, 2])), ("fork", ([1], [7])), ("append", ([7, 1], [1, 1]))]:
        got = getattr(cache, op)(*(ints(*a) for a in args))
        want = getattr(model, op)(*args)
        if op == "append":
            assert got.tolist() == want[0]
        model.check(cache)


def test_append_of_every_length_of_batch(kv):
    for n in (1, 31, 33, 1000, 1025, 4096):
        cache = filled(kv, 1, 2 * n + 3, 16, 1, 8, n, 3)
        model = Model(cache)
        cache.append(torch.arange(n, dtype=torch.int32, device="cuda"), ints(*(1 + i % 20 for i in range(n))))
        model.append(list(range(n)), [1 + i % 20 for i in range(n)])
        model.check(cache)


def test_idle_and_wrong_entries_change_nothing(gpu, kv):
    cache = filled(kv, 1, 20, 16, 1, 64, 6, 4)
    model = Model(cache)
    cache.append(ints(0, -1, 2), ints(20, 9, 5))
    model.append([0, 2], [20, 5])
    model.check(cache)
    cache.free(ints(-1, -5))
    cache.fork(ints(0, 0), ints(-1, 3))
    model.fork([0], [3])
    model.check(cache)
    assert sync_error(gpu) == ""
    for wrong in (lambda: cache.append(ints(6), ints(1)), lambda: cache.append(ints(0, 0), ints(0, 1)),
                  lambda: cache.append(ints(1), ints(-1)), lambda: cache.append(ints(0), ints(4 * 16 - 19)),
                  lambda: cache.free(ints(6)), lambda: cache.fork(ints(0), ints(2)), lambda: cache.fork(ints(6), ints(1)),
                  lambda: cache.fork(ints(-1), ints(1)), lambda: cache.fork(ints(1), ints(1)),
                  lambda: cache.fork(ints(0), ints(6)),
                  lambda: cache.copy(ints(0), ints(20)), lambda: cache.copy(ints(-1), ints(2))):
        wrong()
        assert "outside its cache" in sync_error(gpu)
        model.check(cache)
    # of an entry that comes twice the first counts; a chain of forks is refused where it needs the first
    pos = cache.append(ints(1, 1), ints(3, 4))
    assert pos.tolist() == [0, -1] and "outside its cache" in sync_error(gpu)
    model.append([1], [3])
    cache.fork(ints(0, 0, 4), ints(4, 4, 5))
    assert "outside its cache" in sync_error(gpu)
    model.fork([0], [4])
    model.check(cache)
    cache.free(ints(0, 0), ints(17, 3))
    model.free([0], [3])
    model.check(cache)
    assert sync_error(gpu) == ""


def test_a_shortage_changes_nothing(gpu, kv):
    cache = filled(kv, 1, 5, 16, 1, 64, 3, 6)
    model = Model(cache)
    missing = ints(-1)
    cache.append(ints(0), ints(50))
    model.append([0], [50])
    assert cache.append(ints(1, 0), ints(16, 40), missing=missing).tolist() == [-1, -1] and missing.item() == 2
    model.check(cache)
    assert sync_error(gpu) == ""
    assert cache.append(ints(1), ints(17)).tolist() == [-1]
    assert "too few free pages" in sync_error(gpu)
    model.check(cache)
    assert cache.append(ints(1), ints(16), missing=missing).tolist() == [0] and missing.item() == 0


def test_operations_replay_from_a_graph(kv):
    cache = filled(kv, 2, 64, 16, 2, 64, 8, 8)
    model = Model(cache)
    seqs, prompt, new, missing = ints(0, 1, 2), ints(7, 7, 7), ints(5, 5, 5), ints(0)
    cache.append(ints(7), ints(21))
    model.append([7], [21])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        cache.free(seqs)
        cache.fork(prompt, seqs)
        cache.append(seqs, new, missing)
        live = cache.compact()
    for n in (5, 9, 1):
        new.fill_(n)
        graph.replay()
        model.free([0, 1, 2], [0, 0, 0])
        model.fork([7] * 3, [0, 1, 2])
        model.append([0, 1, 2], [n] * 3)
        assert live.item() == model.compact()
        model.check(cache)


def test_refusals_name_what_is_wrong(gpu, kv):
    lib = gpu.load_cuda()
    cache = filled(kv, 2, 8, 16, 2, 64, 4, 4)
    seqs = ints(0)

    def refused(field, value, word):
        desc = type(cache.desc).from_buffer_copy(cache.desc)
        setattr(desc, field, value)
        assert lib.edgexpu_cuda_kv_free_dev(ctypes.byref(desc), seqs.data_ptr(), None, 1, None) == 0
        assert word in lib.edgexpu_cuda_last_error().decode()

    for field, value, word in [("k", None, "NULL"), ("table", None, "NULL"), ("type", 0, "type 0"), ("page_size", 8, "page size"),
                               ("page_size", 48, "page size"), ("page_size", 512, "page size"), ("head_dim", 12, "head_dim"),
                               ("head_dim", 264, "head_dim"), ("n_pages", 0, "positive"), ("n_seqs", 0, "positive"),
                               ("max_pages", 1 << 28, "2^31"), ("page_stride", 2 * 16 * 64 - 8, "strides"),
                               ("page_stride", 2 * 16 * 64 + 4, "strides"), ("k", cache.desc.k + 8, "aligned")]:
        refused(field, value, word)
    desc = type(cache.desc).from_buffer_copy(cache.desc)
    desc.work = None
    for call in (lambda: lib.edgexpu_cuda_kv_append_dev(ctypes.byref(desc), seqs.data_ptr(), seqs.data_ptr(), 1, None, None, None),
                 lambda: lib.edgexpu_cuda_kv_compact_dev(ctypes.byref(desc), None, None)):
        assert call() == 0 and "work memory" in lib.edgexpu_cuda_last_error().decode()
    assert lib.edgexpu_cuda_kv_append_dev(cache._desc, seqs.data_ptr(), seqs.data_ptr(), 4097, None, None, None) == 0
    assert lib.edgexpu_cuda_kv_fork_dev(cache._desc, None, seqs.data_ptr(), 1, None) == 0
    assert lib.edgexpu_cuda_kv_free_dev(cache._desc, seqs.data_ptr(), None, -1, None) == 0
    assert lib.edgexpu_cuda_kv_free_dev(None, seqs.data_ptr(), None, 1, None) == 0
    with pytest.raises(ValueError):
        cache.append(seqs.long(), seqs)
    with pytest.raises(ValueError):
        cache.append(seqs, ints(1, 2))
    with pytest.raises(ValueError):
        kv.KvCache(cache.k, cache.v.to(torch.bfloat16), cache.table, cache.lens, cache.refs)
    with pytest.raises(ValueError):
        kv.KvCache(cache.k, cache.v, cache.table, cache.lens[:2], cache.refs)
    assert sync_error(gpu) == ""


# ---- norm, rotation and store ------------------------------------------------------------------------


def turned(x, w, eps, rope, pos, halves):
    """x [tokens][heads][dim] in 64 bits: normed and rotated by the table's row of each position."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + eps) * w.double()
    if rope is None:
        return x
    y, rot = x.clone(), rope.shape[1]
    for j in range(rot // 2):
        a, b = (j, j + rot // 2) if halves else (2 * j, 2 * j + 1)
        c, s = (rope[pos, 2 * j + i].double()[:, None] for i in range(2))
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,dim,rot,norm,pairing,n,fused,ps", [
    (9, 3, 64, 64, False, "adjacent", 1, False, 16), (32, 8, 128, 128, True, "halves", 67, True, 64),
    (32, 8, 128, 64, True, "adjacent", 5, False, 16), (4, 4, 256, 256, True, "halves", 3, True, 32),
    (3, 1, 8, 2, True, "adjacent", 9, False, 16), (6, 2, 72, 22, True, "halves", 33, False, 256),
    (2, 1, 104, 0, True, "adjacent", 2, True, 16), (5, 5, 16, 0, False, "halves", 7, False, 16),
    (32, 8, 128, 128, True, "adjacent", 1500, False, 64), (8, 2, 200, 100, False, "halves", 11, True, 128)])
def test_heads_match_the_formulas(gpu, kv, heads, n_kv, dim, rot, norm, pairing, n, fused, ps, dtype):
    torch.manual_seed(n * dim)
    layers, batch, columns = 2, 4, 2 + 600 // ps
    cache = filled(kv, layers, batch * columns, ps, n_kv, dim, batch, columns, DTYPES[dtype], interleaved=fused)
    each = n // batch + 1
    start = [0, 130, 7, 63]
    cache.append(ints(0, 1, 2, 3), ints(*(s + each for s in start)))
    seqs = ints(*([i % batch for i in range(n)] + [-1, 2]))
    pos = ints(*([start[i % batch] + i // batch for i in range(n)] + [3, -1]))
    widths = [heads * dim, n_kv * dim, n_kv * dim]
    rows = torch.randn(n + 2, sum(widths), device="cuda") * torch.rand(n + 2, 1, device="cuda") * 4
    parts = rows.split(widths, 1)
    if not fused:
        parts = [p.contiguous() for p in parts]
    qw, kw = (torch.rand(dim, device="cuda") + 0.5 for _ in range(2)) if norm else (None, None)
    rope = None
    if rot:
        angle = torch.arange(1000, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda") / rot)
        rope = torch.stack([angle.cos(), angle.sin()], -1).reshape(1000, rot).float()
    k0, v0 = cache.k.clone(), cache.v.clone()
    q = cache.qk_norm_rope(1, *parts, seqs, pos, n_heads=heads, q_norm=qw, k_norm=kw, eps=1e-5, rope=rope, pairing=pairing)
    p, live = pos.long().clamp(min=0), torch.arange(n, device="cuda")
    halves = pairing == "halves"
    want_q = turned(parts[0].reshape(n + 2, heads, dim), qw, 1e-5, rope, p, halves)
    want_k = turned(parts[1].reshape(n + 2, n_kv, dim), kw, 1e-5, rope, p, halves)
    want_v = parts[2].reshape(n + 2, n_kv, dim).double()
    # one rounding to the type (2^-11 or 2^-8 of the value; f16 to 2^-25 below its normal range) of an fp32
    # value within 2^-19 of the pair's size: the norm's sum of dim squares, its root and quotient, and
    # two products of the rotation
    unit = 2.0 ** -11 if dtype == "f16" else 2.0 ** -8

    def close(got, want):
        size = want.abs().amax(-1, keepdim=True) * 2.0 ** -19 * 2
        assert bool(((got.double() - want).abs() <= unit * want.abs() + size + 2.0 ** -24).all())

    close(q[:n], want_q[:n])
    assert not q[n:].any()
    page, off = cache.table[seqs[:n].long(), p[:n] // ps].long(), p[:n] % ps
    close(cache.k[1, page, :, off], want_k[:n])
    close(cache.v[1, page, :, off], want_v[:n])
    for pool, before in ((cache.k, k0), (cache.v, v0)):  # nothing else is touched
        pool[1, page, :, off] = before[1, page, :, off]
        assert torch.equal(pool.view(torch.int16), before.view(torch.int16))
    assert sync_error(gpu) == ""


def test_heads_without_a_page_are_errors_and_store_nothing(gpu, kv):
    cache = filled(kv, 1, 8, 16, 1, 64, 3, 4)
    cache.append(ints(0), ints(20))
    before = cache.k.clone()
    x = torch.randn(4, 64, device="cuda")
    rope = torch.ones(18, 64, device="cuda")
    q = cache.qk_norm_rope(0, x, x, x, ints(0, 1, 3, 0), ints(32, 0, 0, 18), n_heads=1, rope=rope)
    assert "outside its cache" in sync_error(gpu)
    assert not q.any() and torch.equal(cache.k, before)
    q = cache.qk_norm_rope(0, x[:1], x[:1], x[:1], ints(0), ints(1 << 30), n_heads=1)
    assert "outside its cache" in sync_error(gpu) and not q.any()
    none = torch.empty(0, 64, device="cuda")
    assert cache.qk_norm_rope(0, none, none, none, ints(), ints(), n_heads=1).shape == (0, 1, 64)
    assert sync_error(gpu) == ""


def test_heads_refusals(gpu, kv):
    cache = filled(kv, 1, 8, 16, 1, 64, 3, 4)
    x = torch.randn(4, 72, device="cuda")
    good, seqs, pos = x[:, :64], ints(0, 0, 0, 0), ints(0, 1, 2, 3)
    for call in (lambda: cache.qk_norm_rope(1, good, good, good, seqs, pos, n_heads=1),
                 lambda: cache.qk_norm_rope(0, x[:, 2:66], good, good, seqs, pos, n_heads=1),
                 lambda: cache.qk_norm_rope(0, good, torch.randn(4, 66, device="cuda")[:, :64], good, seqs, pos, n_heads=1),
                 lambda: cache.qk_norm_rope(0, good, good, good, seqs, pos, n_heads=1, rope=torch.ones(9, 66, device="cuda")),
                 lambda: cache.qk_norm_rope(0, good, good, good, seqs, pos, n_heads=1, rope=torch.ones(9, 7, device="cuda"))):
        with pytest.raises(gpu.EdgexpuError):
            call()
    for call in (lambda: cache.qk_norm_rope(0, good.half(), good, good, seqs, pos, n_heads=1),
                 lambda: cache.qk_norm_rope(0, good, good, good, seqs[:3], pos, n_heads=1),
                 lambda: cache.qk_norm_rope(0, good, good, good, seqs, pos, n_heads=1, q_norm=torch.ones(63, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    assert sync_error(gpu) == ""


def test_heads_of_a_pool_past_32_bit_offsets(kv):
    """The last page of a pool of more than 2^31 elements; its copy, and its move by a packing."""
    pages, ps, dim = 3, 256, 256
    stride = (1 << 31) // 2 + (1 << 20)  # page 2 begins past 2^31 elements
    pools = [torch.zeros(2 * stride + ps * dim, dtype=torch.float16, device="cuda") for _ in range(2)]
    k, v = (torch.as_strided(p, (1, pages, 1, ps, dim), (0, stride, ps * dim, dim, 1)) for p in pools)
    cache = kv.KvCache(k, v, torch.tensor([[2], [-1]], dtype=torch.int32, device="cuda"), ints(256, 0), ints(0, 0, 1))
    x = torch.randn(256, dim, device="cuda")
    cache.qk_norm_rope(0, x, x, 2 * x, torch.zeros(256, dtype=torch.int32, device="cuda"),
                       torch.arange(256, dtype=torch.int32, device="cuda"), n_heads=1)
    want = x.half()
    assert torch.equal(k[0, 2, 0], want) and torch.equal(v[0, 2, 0], (2 * x).half())
    cache.copy(ints(2), ints(1))
    assert torch.equal(k[0, 1, 0], want)
    assert cache.compact().item() == 1 and cache.table.tolist() == [[0], [-1]] and cache.refs.tolist() == [1, 0, 0]
    assert torch.equal(k[0, 0, 0], want) and torch.equal(v[0, 0, 0], (2 * x).half())


def test_a_cache_on_another_device_than_the_librarys_is_refused(gpu, kv):
    assert gpu.load_cuda().edgexpu_cuda_device() == 0
    cache = filled(kv, 1, 4, 16, 1, 8, 2, 2)
    cache.desc.device = 1  # as one that was made before the library was bound
    for call in (lambda: cache.free(ints(0)), lambda: cache.append(ints(0), ints(1)), lambda: cache.compact()):
        with pytest.raises(ValueError, match="the cache is on cuda:1, the library on cuda:0"):
            call()


@pytest.mark.parametrize("n,columns", [(3, 2 ** 27 - 1), (17, 2 ** 27 - 1), (256, 2 ** 23), (512, 2 ** 23), (300, 2 ** 23)])
def test_a_batch_that_asks_for_more_pages_than_32_bits_count(gpu, kv, n, columns):
    """Long rows asked for whole: their sum is 2^31 pages and more, 2^31 and 2^32 among them.  Nothing changes, and
    the pages short are told up to 2^31 - 1."""
    cache = filled(kv, 1, 5, 16, 1, 8, n, columns)
    seqs, whole, missing = torch.arange(n, dtype=torch.int32, device="cuda"), ints(*[16 * columns] * n), ints(-7)
    assert cache.append(seqs, whole, missing=missing).tolist() == [-1] * n
    assert missing.item() == min(n * columns - 5, 2 ** 31 - 1)
    assert not cache.lens.any() and not cache.refs.any() and int(cache.table.max()) == -1
    assert cache.append(ints(0, 1, 2), ints(16, 32, 16), missing=missing).tolist() == [0, 0, 0] and missing.item() == 0
    assert cache.table[:3, :2].tolist() == [[0, -1], [1, 2], [3, -1]]
    assert sync_error(gpu) == ""


def total_of(cache, model, seqs, new):
    """Pages that an append would take."""
    trial = Model(cache)
    trial.rows, trial.lens, trial.refs = [list(r) for r in model.rows], list(model.lens), list(model.refs)
    before = sum(r == 0 for r in trial.refs)
    trial.append(seqs, new)
    return before - sum(r == 0 for r in trial.refs)


@pytest.mark.parametrize("n", [255, 256, 257, 1000, 4096])
@pytest.mark.parametrize("source", [False, True])
def test_append_of_many_forks(gpu, kv, n, source):
    """Rows that share a partly filled last page grow by 0 to 20 tokens, n in a batch: with the row they come from the
    batch holds all of the page's rows, without it not; with idle entries and one that comes twice; and with a page
    too few, where nothing may change."""
    rows = n if source else n + 1
    rng = np.random.default_rng(n + source)
    new = [int(x) for x in rng.choice([0, 1, 5, 20], rows)]
    if source and n < 1000:  # all holders grow, so that one keeps the page
        new = [max(1, x) for x in new]
    seqs = rng.permutation(rows).tolist()
    if not source:
        seqs.remove(0)
    grow = [new[s] for s in seqs]
    probe = filled(kv, 1, 3 * rows + 4, 16, 1, 8, rows, 4)
    model = Model(probe)
    model.append([0], [21])
    model.fork([0] * (rows - 1), list(range(1, rows)))
    need = total_of(probe, model, seqs, grow) + 2
    for short in (1, 0):
        cache = filled(kv, 1, need - short, 16, 1, 8, rows, 4)
        model = Model(cache)
        cache.append(ints(0), ints(21))
        model.append([0], [21])
        cache.fork(ints(*[0] * (rows - 1)), ints(*range(1, rows)))
        model.fork([0] * (rows - 1), list(range(1, rows)))
        model.check(cache)
        missing = ints(9)
        got = cache.append(ints(*seqs), ints(*grow), missing=missing).tolist()
        pos, lack = model.append(seqs, grow)
        assert (got, missing.item()) == (pos, lack) and lack == short
        model.check(cache)
    assert sync_error(gpu) == ""
    if n < 4096:  # an idle entry and one that comes twice, of which the first counts
        cache = filled(kv, 1, need + 3 * rows, 16, 1, 8, rows, 4)
        model = Model(cache)
        cache.append(ints(0), ints(21))
        model.append([0], [21])
        cache.fork(ints(*[0] * (rows - 1)), ints(*range(1, rows)))
        model.fork([0] * (rows - 1), list(range(1, rows)))
        twice = seqs[n // 2]
        got = cache.append(ints(-1, *seqs, twice), ints(7, *grow, 3)).tolist()
        assert got == [-1] + model.append(seqs, grow)[0] + [-1]
        model.check(cache)
        assert "outside its cache" in sync_error(gpu)
        got = cache.append(ints(*seqs), ints(*[1] * n)).tolist()  # rows that are apart by now, and those that are not
        assert got == model.append(seqs, [1] * n)[0]
        model.check(cache)
        assert sync_error(gpu) == ""


def test_synchronize_raises_what_the_device_found(gpu, kv):
    cache = filled(kv, 1, 4, 16, 1, 64, 2, 6)
    x = torch.randn(1, 64, device="cuda")
    cache.synchronize()
    for call, word in [(lambda: cache.append(ints(0), ints(80)), "too few free pages"), (lambda: cache.free(ints(2)), "outside its cache"),
                       (lambda: cache.qk_norm_rope(0, x, x, x, ints(1), ints(0), n_heads=1), "outside its cache"),
                       (lambda: cache.attention(0, x.half().reshape(1, 1, 64), ints(7)), "outside its cache")]:
        for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
            with torch.cuda.stream(stream):
                call()
                with pytest.raises(gpu.EdgexpuError, match=word):
                    cache.synchronize()
                cache.synchronize()  # told once
