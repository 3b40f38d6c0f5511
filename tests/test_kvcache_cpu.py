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


def test_calls_without_a_device_fail(cuda):
    import torch

    if torch.cuda.is_available():
        pytest.skip("checks the no-device failure path")
    pkg = load_pkg()
    desc = pkg.KvCacheDesc()
    assert cuda.edgexpu_cuda_kv_free_dev(ctypes.byref(desc), None, None, 0, None) == 0
    assert cuda.edgexpu_cuda_last_error()
    assert cuda.edgexpu_cuda_kv_attention_dev(ctypes.byref(desc), 0, None, None, None, 1, 1, 1, 0, 0, 1, 1.0, None, 1, None, 0, None) == 0
