"""The paged cache's host side without a device: sizes, and refusals before any launch."""

import ctypes

import pytest

from _oracle import load_pkg


@pytest.fixture(scope="module")
def cuda():
    pkg = load_pkg()
    if not pkg.CUDA_LIB.exists():
        pytest.skip("library not built")
    return pkg.load_cuda()


def test_work_bytes(cuda):
    f = cuda.edgexpu_cuda_kv_work_bytes
    assert f(0, 4) == 0 and f(4, 0) == 0
    assert f(100, 7) == (16 + 4 * 7 + 3 * 100) * 4
    assert f(2**31 - 1, 1) > 3 * 4 * (2**31 - 1)  # no overflow


def test_descriptor_matches_the_header():
    pkg = load_pkg()
    d = pkg.KvCacheDesc
    assert ctypes.sizeof(d) == 96
    assert (d.layer_stride.offset, d.type.offset, d.n_layers.offset, d.max_pages.offset, d.table.offset, d.work.offset) == (
        16, 32, 36, 60, 64, 88)


def test_attention_work_bytes(cuda):
    pkg = load_pkg()

    def need(batch, tokens, heads, shared, longest, n_kv=8, dim=128):
        desc = pkg.KvCacheDesc(n_kv=n_kv, head_dim=dim)
        return cuda.edgexpu_cuda_kv_attention_work_bytes(ctypes.byref(desc), batch, tokens, heads, shared, longest)

    assert need(1, 1, 30, 0, 100) == 0  # heads not a multiple of the key heads
    assert need(0, 0, 32, 0, 100) == 0 and need(1, 1, 32, 0, 0) == 0
    row = 32 * (128 * 4 + 8)
    assert need(4, 4, 32, 4096, 8192) >= 2 * 4 * row  # at least a part of the prefix and one of the own positions
    # grows with the tokens, and stays far from the keys and values' own size
    assert need(128, 128, 32, 32768, 34768) < 64 * 128 * row
    assert need(2**31 - 1, 2**31 - 1, 8, 0, 1) >= 0
    assert cuda.edgexpu_cuda_kv_attention_work_bytes(None, 1, 1, 1, 0, 1) == 0


def test_attention_work_bytes_before_the_library_is_bound(cuda):
    """128 single tokens on up to 32000 positions of their own: the line of tiles is cut for a B200's SMs, 16 rows
    that continue an earlier block's run for each block, at least one block an SM."""
    pkg = load_pkg()
    desc = pkg.KvCacheDesc(n_kv=8, head_dim=128)
    need = cuda.edgexpu_cuda_kv_attention_work_bytes(ctypes.byref(desc), 128, 128, 32, 0, 32000)
    assert need >= (128 * 32 + 16 * 148) * (128 * 4 + 8)


def test_single_tokens_pieces_stay_short_where_the_shared_pass_leaves_few_sms(cuda):
    """128 single tokens behind 32k, 148 SMs: the shared pass takes all of them with up to 192 own positions and all but
    two with 224 and 256; the own pass's blocks get 16 tiles at most all the same, or there are four an SM."""
    pkg = load_pkg()
    desc = pkg.KvCacheDesc(n_kv=8, head_dim=128)
    slot = 128 * 32  # rows of a part: tokens x heads

    def rows(own):
        size = cuda.edgexpu_cuda_kv_attention_work_bytes(ctypes.byref(desc), 128, 128, 32, 32768, 32768 + own)
        up = lambda n: (n + 255) // 256 * 256  # noqa: E731
        return next(r for r in range(size // 520, 0, -1) if up(r * 8) + up(r * 512) + up(129 * 4) == size)

    # as many parts with 224 and 256, for 72 to 74 pieces of a line of 8
    parts = (rows(192) - 16 * 4 * 148) // slot
    assert parts * slot + 16 * 4 * 148 == rows(192)
    for own in (224, 256):
        tiles = 128 * 8 * ((own + 63) // 64 + 1)
        blocks = (rows(own) - parts * slot) // 16
        assert blocks >= min(4 * 148, tiles // 16), (own, blocks, tiles)


def test_calls_without_a_device_fail(cuda):
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-device failure path")
    pkg = load_pkg()
    desc = pkg.KvCacheDesc()
    assert cuda.edgexpu_cuda_kv_free_dev(ctypes.byref(desc), None, None, 0, None) == 0
    assert cuda.edgexpu_cuda_last_error()
    assert cuda.edgexpu_cuda_kv_attention_dev(ctypes.byref(desc), 0, None, None, None, 1, 1, 1, 0, 0, 1, 1.0, None, 1, None, 0, None) == 0


@pytest.fixture(scope="module")
def kv():
    pkg = load_pkg()
    pytest.importorskip("torch")
    if not (pkg.LIB_DIR / "_kv_torch.so").exists():
        pytest.skip("torch module not built")
    from edgexpu_llm_b200 import kv as module

    return module


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
def test_tensors_of_another_device_are_refused(kv):
    """Each argument in turn on another GPU than the cache's, or on the host: a ValueError before any launch.  The
    tensors are stand-ins that have a device and no memory, so none is needed here."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    if torch.cuda.device_count() == 1:
        pytest.skip("a stand-in for a second GPU needs two where there is one")
    with FakeTensorMode():
        cache = kv.KvCache.empty(1, 4, 16, 1, 8, 3, 2, device="cuda:0")

        def ints(n):
            return torch.zeros(n, dtype=torch.int32, device="cuda:0")

        def rows(n):
            return torch.zeros(n, 8, device="cuda:0")

        half = torch.zeros(2, 1, 8, dtype=torch.float16, device="cuda:0")
        calls = [(cache.append, [ints(2), ints(2), ints(1)], {}), (cache.fork, [ints(2), ints(2)], {}),
                 (cache.free, [ints(2), ints(2)], {}), (cache.copy, [ints(2), ints(2)], {}),
                 (cache.qk_norm_rope, [0, rows(2), rows(2), rows(2), ints(2), ints(2), 1],
                  dict(q_norm=rows(1)[0], k_norm=rows(1)[0], rope=rows(9), out=half)),
                 (cache.attention, [0, half, ints(2)], dict(q_start=ints(3), out=half))]
        for device in ("cuda:1", "cpu"):
            for call, args, named in calls:
                for at, x in list(enumerate(args)) + list(named.items()):
                    if not isinstance(x, torch.Tensor):
                        continue
                    a, k = list(args), dict(named)
                    (k if isinstance(at, str) else a)[at] = x.to(device)
                    with pytest.raises(ValueError, match=r"on cuda:0; got .* on " + device):
                        call(*a, **k)


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
def test_a_cache_is_made_on_the_librarys_device_alone(kv, monkeypatch):
    from torch._subclasses.fake_tensor import FakeTensorMode

    class Library:
        def __init__(self, device):
            self.edgexpu_cuda_device = lambda: device
            self.edgexpu_cuda_kv_work_bytes = lambda pages, seqs: 64

    with FakeTensorMode():
        for bound in (-1, 0):
            monkeypatch.setattr(kv, "load_cuda", lambda: Library(bound))
            kv.KvCache.empty(1, 4, 16, 1, 8, 2, 2, device="cuda:0")
        monkeypatch.setattr(kv, "load_cuda", lambda: Library(1))
        with pytest.raises(ValueError, match="the cache is on cuda:0, the library on cuda:1"):
            kv.KvCache.empty(1, 4, 16, 1, 8, 2, 2, device="cuda:0")


def test_device_of_an_unbound_library(cuda):
    import torch

    if torch.cuda.is_available():
        pytest.skip("another test may have bound it")
    assert cuda.edgexpu_cuda_device() == -1
