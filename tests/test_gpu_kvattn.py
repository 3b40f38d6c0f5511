"""Attention over the paged cache against the formula in 64 bits.

Tolerance of an output of a row with softmax weights p and values v, u the type's unit roundoff (2^-11 for
f16, 2^-8 for bf16): u sum p|v| for the weights rounded to the type, 2^-15 sum p|v| for fp32 sums, scores and
exponentials (a score of dim products is off by at most dim 2^-23 of the sum of their sizes, about 2^-17 of a
weight for the standard normal heads here), and u |out| + 2^-24 for the output's own rounding, where it has one.
"""

import ctypes
import pathlib
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def kv(gpu):
    from edgexpu_llm_b200 import kv as module

    return module


def sync_error(gpu):
    buf = ctypes.create_string_buffer(512)
    ok = gpu.load_cuda().edgexpu_cuda_stream_sync(torch.cuda.current_stream().cuda_stream, buf, 512)
    return "" if ok else buf.value.decode()


def ints(*v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def make(kv, lens, shared, heads, n_kv, dim, ps, dtype, layers=1, seed=0, slack=float("nan")):
    """A cache with row 0 the prefix and rows 1 .. the sequences (their first `shared` positions its pages, or
    copies where a page is not full), pages in random order, and `slack` wherever no token is."""
    gen = torch.Generator().manual_seed(seed)
    full = shared // ps
    counts = [-(-shared // ps)] + [max(0, -(-n // ps) - full) for n in lens]
    pages, columns = sum(counts) + 3, max(1, max(-(-n // ps) for n in [shared] + list(lens)) + 1)
    order = torch.randperm(pages, generator=gen).tolist()
    table, at = torch.full((len(lens) + 1, columns), -1, dtype=torch.int32), 0
    for i, (n, c) in enumerate(zip([shared] + list(lens), counts)):
        mine = order[at:at + c]
        at += c
        row = mine if i == 0 else (table[0, :full].tolist() + mine)[: -(-n // ps)]
        table[i, : len(row)] = torch.tensor(row, dtype=torch.int32)
    shape = (layers, pages, n_kv, ps, dim)
    k, v = (torch.full(shape, slack, dtype=dtype, device="cuda") for _ in range(2))
    torch.manual_seed(seed)
    total = max([shared] + list(lens))
    for i, n in enumerate([shared] + list(lens)):
        data = torch.randn(2, layers, n_kv, n, dim, device="cuda").to(dtype)
        if i == 0:
            prefix = data
        else:
            data[:, :, :, : min(n, shared)] = prefix[:, :, :, : min(n, shared)]
        for p in range(0, n, ps):
            page, m = int(table[i, p // ps]), min(ps, n - p)
            k[:, page, :, :m], v[:, page, :, :m] = data[0, :, :, p:p + m], data[1, :, :, p:p + m]
    del total
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).int()
    return kv.KvCache(k, v, table.cuda(), ints(shared, *lens), refs.cuda())


def reference(cache, layer, q, seqs, starts, scale):
    """(out, sum of p|v|) of every token and head in 64 bits."""
    ps, dim = cache.k.shape[3:]
    n_kv, rep = cache.k.shape[2], q.shape[1] // cache.k.shape[2]
    out, size = (torch.zeros(q.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for i, s in enumerate(seqs):
        a, b = starts[i], starts[i + 1]
        n = int(cache.lens[s]) if s >= 0 else 0
        if n == 0:
            continue
        pages = cache.table[s, : -(-n // ps)].long()
        k, v = (x[layer, pages].double().transpose(0, 1).reshape(n_kv, -1, dim)[:, :n].repeat_interleave(rep, 0) for x in (cache.k, cache.v))
        for t in range(a, b):
            vis = n - (b - a) + (t - a) + 1
            if vis > 0:
                score = torch.einsum("hd,hjd->hj", q[t].double(), k[:, :vis]) * scale
                p = torch.softmax(score, -1)
                out[t] = torch.einsum("hj,hjd->hd", p, v[:, :vis])
                size[t] = torch.einsum("hj,hjd->hd", p, v[:, :vis].abs())
    return out, size


def check(cache, got, layer, q, seqs, starts, scale):
    want, size = reference(cache, layer, q, seqs, starts, scale)
    u = UNIT[q.dtype]
    bound = (u + 2.0 ** -15) * size + (u * want.abs() + 2.0 ** -24 if got.dtype != torch.float32 else 0) + 1e-30
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{int(bad.sum())} outside, worst {float((err / bound).max()):.2f} of the bound, at {bad.nonzero()[:4].tolist()}"


def run(kv, lens, shared, heads, n_kv, dim, ps, dtype, n_q=None, seqs=None, layers=1, out_dtype=None, max_len=None, seed=0, scale=None):
    cache = make(kv, lens, shared, heads, n_kv, dim, ps, DTYPES[dtype], layers, seed)
    seqs = list(range(1, len(lens) + 1)) if seqs is None else seqs
    count = n_q or [1] * len(seqs)
    starts = [sum(count[:i]) for i in range(len(count) + 1)]
    q = torch.randn(starts[-1], heads, dim, device="cuda").to(DTYPES[dtype])
    scale = dim ** -0.5 if scale is None else scale
    got = cache.attention(layers - 1, q, ints(*seqs), q_start=ints(*starts) if n_q else None, shared_seq=0, shared_len=shared,
                          max_len=max_len, scale=scale, out_dtype=out_dtype)
    check(cache, got, layers - 1, q, seqs, starts, scale)
    return cache, q, got


# one token: lengths around tiles, pages and parts; every head layout
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,dim", [(9, 3, 64), (32, 8, 128), (1, 1, 8), (12, 2, 96), (40, 1, 128), (4, 4, 256), (7, 1, 72),
                                            (34, 2, 64), (130, 1, 128)])
@pytest.mark.parametrize("ps", [16, 64, 256])
def test_single_tokens(gpu, kv, heads, n_kv, dim, ps, dtype):
    run(kv, [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 1000], 0, heads, n_kv, dim, ps, dtype, seed=heads * dim)
    assert sync_error(gpu) == ""


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shared,ps,heads,n_kv,dim", [
    (1, 16, 9, 3, 64), (15, 16, 32, 8, 128), (64, 16, 32, 8, 128), (65, 64, 12, 2, 96), (127, 32, 32, 8, 128), (128, 128, 4, 4, 256),
    (1000, 64, 32, 8, 128), (4097, 64, 32, 8, 128), (4097, 16, 9, 3, 64), (2050, 16, 40, 1, 128), (700, 256, 16, 2, 80)])
@pytest.mark.parametrize("batch", [1, 5, 40])
def test_single_tokens_behind_a_prefix(gpu, kv, batch, shared, ps, heads, n_kv, dim, dtype):
    lens = [shared + 1 + (i * 97) % 200 for i in range(batch)]
    run(kv, lens, shared, heads, n_kv, dim, ps, dtype, seed=shared)
    assert sync_error(gpu) == ""


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,dim,ps", [(9, 3, 64, 16), (32, 8, 128, 64), (12, 2, 96, 16), (4, 4, 256, 32)])
@pytest.mark.parametrize("shared,n_q,more", [
    (0, [1, 2, 3], [0, 0, 5]), (0, [70, 1, 0, 33], [0, 3, 9, 100]), (100, [5, 64, 1], [0, 0, 30]), (513, [17, 0, 200, 4], [1, 1, 1, 90]),
    (2000, [130, 129], [0, 64])])
def test_several_tokens(gpu, kv, shared, n_q, more, heads, n_kv, dim, ps, dtype):
    run(kv, [shared + a + b for a, b in zip(n_q, more)], shared, heads, n_kv, dim, ps, dtype, n_q=n_q, seed=shared)
    assert sync_error(gpu) == ""


def test_many_tokens_of_one_sequence(kv):
    run(kv, [1500], 0, 32, 8, 128, 64, "bf16", n_q=[1500])
    run(kv, [900], 300, 8, 8, 64, 16, "f16", n_q=[600])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_sequences_that_do_not_reach_past_the_prefix(gpu, kv, dtype):
    """Lengths inside the prefix, its very end, and tokens of which some see less than all of it."""
    run(kv, [1, 77, 199, 200, 201, 260], 200, 8, 2, 64, 16, dtype)
    run(kv, [203, 190, 200, 230, 40], 200, 8, 2, 64, 16, dtype, n_q=[5, 3, 1, 30, 40])
    assert sync_error(gpu) == ""


def test_idle_entries_and_empty_rows_give_zero(gpu, kv):
    for n_q in (None, [1, 3, 2, 0, 4]):
        cache = make(kv, [50, 0, 2, 9], 0, 4, 2, 64, 16, torch.float16)
        seqs = [1, -1, 2, -1, 3]  # the second sequence is empty; the third is shorter than its four tokens
        starts = [0, 1, 2, 3, 4, 5] if n_q is None else [0, 1, 4, 6, 6, 10]
        q = torch.randn(starts[-1], 4, 64, device="cuda").half()
        out = torch.full_like(q, 7.0)
        for shared, max_len in ((0, 50), (0, 6400)):
            cache.attention(0, q, ints(*seqs), q_start=None if n_q is None else ints(*starts), shared_len=shared, max_len=max_len, out=out)
            check(cache, out, 0, q, seqs, starts, 64 ** -0.5)
            assert not out[starts[1]:starts[4]].any()
    run(kv, [40, 30, 25], 20, 4, 2, 64, 16, "f16", seqs=[3, -1, 1, 1, -1])
    run(kv, [40, 30, 25], 20, 4, 2, 64, 16, "f16", seqs=[-1, -1])
    assert sync_error(gpu) == ""


def test_fp32_output_layers_and_length_hints(kv):
    for dtype in ("f16", "bf16"):
        a = run(kv, [300, 20, 777], 0, 32, 8, 128, 64, dtype, out_dtype=torch.float32, layers=3)
        for hint in (1, 20, 777, 100000):  # the hint divides the work, no more
            run(kv, [300, 20, 777], 128, 32, 8, 128, 64, dtype, out_dtype=torch.float32, max_len=hint, seqs=[1, 3])
        assert a[2].dtype == torch.float32


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0, 30.0])
def test_scales(kv, scale):
    """A softmax that is flat, upside down or all but a maximum."""
    for dtype in ("f16", "bf16"):
        cache = make(kv, [500, 40], 100, 8, 2, 64, 16, DTYPES[dtype])
        q = (torch.randn(2, 8, 64, device="cuda") * 0.2).to(DTYPES[dtype])
        got = cache.attention(0, q, ints(1, 2), shared_len=40, scale=scale)
        want, size = reference(cache, 0, q, [1, 2], [0, 1, 2], scale)
        # a score of size up to 30 * 8 is off by 2^-17 of that at most, and a weight by twice as much
        bound = (2 * UNIT[q.dtype] + 2.0 ** -15 + 2.0 ** -16 * abs(scale) * 16) * size + 2.0 ** -24
        assert bool(((got.double() - want).abs() <= bound).all())


def test_a_large_score_beside_many_small_ones(kv):
    """Weights far below f16's smallest still add up: one position at weight 1, 20000 at about 2^-20."""
    cache = make(kv, [20001], 0, 1, 1, 64, 64, torch.float16)
    pages = cache.table[1, :313].long()
    cache.k[0, pages] = 0
    cache.v[0, pages] = 0
    cache.k[0, pages[0], 0, 3, 0] = 14.0
    cache.v[0, pages, :, :, 1] = 1.0
    cache.v[0, pages[0], 0, 3, 1] = 0.0
    q = torch.zeros(1, 1, 64, device="cuda").half()
    q[..., 0] = 1.0
    got = cache.attention(0, q, ints(1), scale=1.0, out_dtype=torch.float32)
    want, size = reference(cache, 0, q, [1], [0, 1], 1.0)
    assert bool(((got.double() - want).abs() <= (2.0 ** -11 + 2.0 ** -15) * size + 1e-9).all())


def test_infinities_and_nan_of_the_data(kv):
    """What a token sees decides alone: a NaN or infinity it sees spreads as in the formula, one it does not
    see is as nothing, in keys and in values, in other heads, later tokens and other sequences."""
    for n_q in (None, [1, 12, 3]):
        starts = [0, 1, 2, 3] if n_q is None else [0, 1, 13, 16]
        cache = make(kv, [130, 140, 90], 64, 4, 2, 64, 16, torch.bfloat16)
        t = cache.table.long()
        cache.v[0, t[2, 133 // 16], 0, 133 % 16, 5] = float("inf")   # sequence 2, position 133, kv head 0
        cache.v[0, t[2, 136 // 16], 1, 136 % 16, 9] = float("nan")
        cache.k[0, t[2, 138 // 16], 1, 138 % 16, 2] = float("nan")
        cache.k[0, t[3, 70 // 16], 0, 70 % 16] = float("-inf")
        q = torch.randn(starts[-1], 4, 64, device="cuda").bfloat16().abs()
        got = cache.attention(0, q, ints(1, 2, 3), q_start=None if n_q is None else ints(*starts), shared_len=64)
        want, size = reference(cache, 0, q, [1, 2, 3], starts, 0.125)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
        fine = want.isfinite() & size.isfinite()
        u = 2.0 ** -8
        assert bool(((got.double() - want).abs() <= (u + 2.0 ** -15) * size + u * want.abs())[fine].all())
        if n_q is not None:
            assert not want[1:6].isnan().any() and want[8:13].isnan().any()
    # in the prefix too, with few rows and with many
    for batch in (1, 3, 20, 90):
        cache = make(kv, [210] * batch, 200, 4, 2, 64, 16, torch.float16)
        t = cache.table.long()
        for x, value in ((7, float("inf")), (50, float("-inf")), (199, float("inf"))):
            cache.v[0, t[0, x // 16], 0, x % 16, x % 61] = value
        cache.v[0, t[1:, 199 // 16], 0, 199 % 16, 199 % 61] = float("inf")  # the copies of the page it shares in part
        cache.k[0, t[0, 3], 1, 2, 4] = float("nan")
        q = torch.randn(batch, 4, 64, device="cuda").half()
        got = cache.attention(0, q, ints(*range(1, batch + 1)), shared_len=200)
        want, _ = reference(cache, 0, q, list(range(1, batch + 1)), list(range(batch + 1)), 0.125)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isposinf(), want.isposinf())
        assert torch.equal(got.isneginf(), want.isneginf()) and want.isinf().any() and want.isfinite().any()
    # a row all of whose scores are -inf is 0/0
    cache = make(kv, [40], 0, 1, 1, 64, 16, torch.float16)
    cache.k[0, cache.table[1, :3].long()] = float("-inf")
    q = torch.ones(1, 1, 64, device="cuda").half()
    assert cache.attention(0, q, ints(1)).isnan().all()


def test_strided_pools_and_offsets_past_32_bits(gpu, kv):
    pages, ps, dim = 3, 64, 128
    stride = (1 << 31) // 2 + (1 << 20)
    pools = [torch.empty(2 * stride + 2 * ps * dim, dtype=torch.float16, device="cuda") for _ in range(2)]
    k, v = (torch.as_strided(p, (1, pages, 2, ps, dim), (0, stride, ps * dim, dim, 1)) for p in pools)
    k.normal_()
    v.normal_()
    cache = kv.KvCache(k, v, torch.tensor([[2, 0], [2, 1]], dtype=torch.int32, device="cuda"), ints(64, 100), ints(1, 1, 2))
    q = torch.randn(2, 4, dim, device="cuda").half()
    for shared in (0, 64):
        got = cache.attention(0, q, ints(1, 1), shared_len=shared)
        check(cache, got, 0, q, [1, 1], [0, 1, 2], dim ** -0.5)
    both = torch.randn(2, 9, 2, 2, 16, 64, device="cuda").half()  # k and v side by side in one buffer
    cache = kv.KvCache(both[:, :, 0], both[:, :, 1], torch.tensor([[7, 1, 4], [7, 3, 8]], dtype=torch.int32, device="cuda"),
                       ints(16, 41), torch.ones(9, dtype=torch.int32, device="cuda"))
    q = torch.randn(1, 6, 64, device="cuda").half()
    check(cache, cache.attention(1, q, ints(1), shared_len=16), 1, q, [1], [0, 1], 0.125)
    assert sync_error(gpu) == ""


def test_wrong_tables_are_errors_without_a_fault(gpu, kv):
    for n_q, shared in ((None, 0), (None, 32), ([40, 1], 32)):
        cache = make(kv, [90, 70], 32, 4, 2, 64, 16, torch.float16)
        starts = ints(0, 1, 2) if n_q is None else ints(0, 40, 41)
        q = torch.randn(2 if n_q is None else 41, 4, 64, device="cuda").half()
        args = dict(q_start=None if n_q is None else starts, shared_len=shared)
        cache.attention(0, q, ints(1, 2), **args)
        assert sync_error(gpu) == ""
        cache.attention(0, q, ints(1, 3), **args)
        assert "outside its cache" in sync_error(gpu)
        for value in (-1, 10 ** 6):
            was = cache.table.clone()
            cache.table[1, 1 if shared == 0 else 3] = value
            cache.table[0, 1] = value
            cache.attention(0, q, ints(1, 2), **args)
            assert "outside its cache" in sync_error(gpu)
            cache.table.copy_(was)
        cache.lens[2] = 10 ** 6
        cache.attention(0, q, ints(1, 2), **args)
        assert "outside its cache" in sync_error(gpu)
    for starts in ([0, 50, 41], [-3, 40, 41], [0, 10 ** 9, 41]):
        cache.lens[2] = 70
        cache.attention(0, q, ints(1, 2), q_start=ints(*starts), shared_len=32)
        assert "outside its cache" in sync_error(gpu)


def test_streams_and_graphs(gpu, kv):
    cache = make(kv, [100 + i for i in range(8)], 64, 32, 8, 128, 64, torch.float16)
    q, seqs = torch.randn(8, 32, 128, device="cuda").half(), ints(*range(1, 9))
    want = cache.attention(0, q, seqs, shared_len=64, max_len=128)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        outs = [cache.attention(0, q, seqs, shared_len=64, max_len=128) for _ in range(5)]
    outs += [cache.attention(0, q, seqs, shared_len=64, max_len=128) for _ in range(5)]
    torch.cuda.synchronize()
    for o in outs:  # fixed order of every sum: the same bits, on any stream
        assert torch.equal(o, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attention(0, q, seqs, shared_len=64, max_len=128)
    for n in (70, 64, 90):
        cache.lens[1:] = n
        graph.replay()
        check(cache, out, 0, q, list(range(1, 9)), list(range(9)), 128 ** -0.5)
    assert sync_error(gpu) == ""


def test_refusals(gpu, kv):
    cache = make(kv, [40, 50], 16, 4, 2, 64, 16, torch.float16)
    q, seqs = torch.randn(2, 4, 64, device="cuda").half(), ints(1, 2)
    lib = gpu.load_cuda()
    work = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    good = [cache._desc, 0, q.data_ptr(), seqs.data_ptr(), None, 2, 2, 4, 0, 16, 64, 0.125, out.data_ptr(), gpu.TYPE_F16,
            work.data_ptr(), 1 << 20, None]
    assert lib.edgexpu_cuda_kv_attention_dev(*good) == 1
    for at, value, word in [(0, None, "NULL"), (1, 1, "layer 1"), (1, -1, "layer"), (2, None, "invalid"), (2, q.data_ptr() + 2, "aligned"),
                            (3, None, "invalid"), (5, 3, "entries"), (7, 3, "heads"), (7, 0, "heads"), (8, 3, "shared sequence"),
                            (8, -1, "shared sequence"), (10, 0, "max_len"), (12, None, "invalid"), (12, out.data_ptr() + 4, "aligned"),
                            (13, gpu.TYPE_BF16, "output type"), (14, None, "work memory"), (14, work.data_ptr() + 8, "work memory"),
                            (15, 16, "work memory"), (6, -1, "tokens"), (5, -1, "entries")]:
        call = list(good)
        call[at] = value
        assert lib.edgexpu_cuda_kv_attention_dev(*call) == 0, (at, value)
        assert word in lib.edgexpu_cuda_last_error().decode(), (at, value, lib.edgexpu_cuda_last_error())
    assert cache.attention(0, q[:0], ints()).shape == (0, 4, 64)
    for call in (lambda: cache.attention(0, q.bfloat16(), seqs), lambda: cache.attention(0, q[:, :, :32], seqs),
                 lambda: cache.attention(0, q, seqs.long()), lambda: cache.attention(0, q, seqs, q_start=ints(0, 1))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(gpu.EdgexpuError):
        cache.attention(0, q, seqs, out_dtype=torch.bfloat16)
    assert sync_error(gpu) == ""


@pytest.mark.parametrize("scale", [0.0, -0.1, 30.0])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,dim,ps,batch", [(8, 2, 64, 16, 10), (32, 8, 128, 64, 40), (12, 2, 96, 16, 50), (4, 4, 256, 32, 30)])
@pytest.mark.parametrize("shared", [100, 130, 192])
def test_scales_of_many_rows(kv, shared, heads, n_kv, dim, ps, batch, dtype, scale):
    """As test_scales, with 30 to 300 rows of a key head against a prefix that ends in a tile's first half, in its
    second, or with it: blocks of 128 and of 256 rows, and the wide heads' kernel."""
    cache = make(kv, [shared + 1 + i % 70 for i in range(batch)], shared, heads, n_kv, dim, ps, DTYPES[dtype])
    q = (torch.randn(batch, heads, dim, device="cuda") * 0.2).to(DTYPES[dtype])
    seqs = list(range(1, batch + 1))
    got = cache.attention(0, q, ints(*seqs), shared_len=shared, scale=scale)
    want, size = reference(cache, 0, q, seqs, list(range(batch + 1)), scale)
    # dim products of 0.2 normals and normals: sizes add up to 48 at most, a score is off by 2^-17 of that, a weight
    # (and the sum that divides it) by as much
    bound = (2 * UNIT[q.dtype] + 2.0 ** -15 + 2.0 ** -16 * abs(scale) * 48) * size + 2.0 ** -24
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,dim,ps,shared,n_q,own", [
    (32, 8, 128, 64, 1000, None, 33), (32, 8, 128, 64, 700, [64, 1, 17, 40], 3), (9, 3, 64, 16, 300, [100, 50], 0),
    (12, 2, 96, 16, 0, [70, 33], 20), (4, 4, 256, 32, 500, [30, 70], 5), (34, 2, 64, 16, 0, None, 900)])
def test_fp32_output_keeps_the_weights_to_16_bits_and_more(kv, heads, n_kv, dim, ps, shared, n_q, own, dtype):
    """fp32 out: the weights go to their product in two numbers of the type, whichever kernel makes it, so that they
    are off by 2^-15 (bf16) or 2^-20 (f16), or by 2^-33 of the row's largest; sums, scores and exponentials as above."""
    count = n_q or [1] * 70
    lens = [shared + n + own + i % 50 for i, n in enumerate(count)]
    cache = make(kv, lens, shared, heads, n_kv, dim, ps, DTYPES[dtype], seed=dim)
    starts = [sum(count[:i]) for i in range(len(count) + 1)]
    q = torch.randn(starts[-1], heads, dim, device="cuda").to(DTYPES[dtype])
    seqs = list(range(1, len(lens) + 1))
    got = cache.attention(0, q, ints(*seqs), q_start=ints(*starts) if n_q else None, shared_len=shared, scale=dim ** -0.5,
                          out_dtype=torch.float32)
    want, size = reference(cache, 0, q, seqs, starts, dim ** -0.5)
    weights = 2.0 ** -15 if dtype == "bf16" else 2.0 ** -20
    bound = (weights + 2.0 ** -15) * size + max(lens) * 2.0 ** -33 * 6  # values of at most 6
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def test_work_bytes_are_the_same_before_and_after_init():
    code = """
import ctypes, itertools, sys
sys.path.insert(0, {tests!r})
from _oracle import load_pkg
pkg = load_pkg()
f = pkg.load_cuda().edgexpu_cuda_kv_attention_work_bytes
def sizes():
    return [f(ctypes.byref(pkg.KvCacheDesc(n_kv=n_kv, head_dim=dim)), batch, batch * each, 4 * n_kv, shared, shared + more)
            for n_kv, dim, batch, each, shared, more in itertools.product((1, 8), (64, 128, 256), (1, 30, 128, 1100), (1, 7), (0, 100, 32768), (1, 700, 20000))]
before = sizes()
pkg.init(0)
assert sizes() == before
pkg.shutdown()
"""
    subprocess.run([sys.executable, "-c", code.format(tests=str(pathlib.Path(__file__).parent))], check=True, timeout=300)


@pytest.mark.parametrize("n_q,batch", [(None, 160), ([300], 1)])
def test_more_blocks_of_rows_than_half_the_sms(kv, n_q, batch):
    """130 heads on one key head: 78 blocks of 256 rows and more, which then go along the prefix one after the other."""
    lens = [200 + (n_q[0] if n_q else 1) + i % 40 for i in range(batch)]
    run(kv, lens, 200, 130, 1, 64, 16, "bf16", n_q=n_q)
    run(kv, lens, 200, 130, 1, 128, 64, "f16", n_q=n_q, out_dtype=torch.float32)


@pytest.mark.parametrize("batch", [1023, 1024, 1025, 1100])
def test_a_thousand_single_tokens(kv, batch):
    """Around the number of entries up to which single tokens have a kernel of their own."""
    for shared, more in ((0, 40), (70, 1), (70, 130)):
        run(kv, [shared + more + i % 30 for i in range(batch)], shared, 2, 1, 64, 16, "f16", max_len=shared + more + 700)
