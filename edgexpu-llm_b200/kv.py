"""A key/value cache in pages that many sequences share, on torch tensors.

:class:`KvCache` binds the ``edgexpu_cuda_kv_*`` and ``edgexpu_cuda_qk_norm_rope_dev`` calls of
``include/edgexpu_cuda.h``, which say what each call does.  Tensors live on the library's device and
calls run on torch's current stream; none of them waits for the device.  A tensor of another type, shape
or device is a ValueError, a call that the library refuses an EdgexpuError.  What only the device finds (a
sequence or page outside its cache, too few free pages, a wait that ran out) is an EdgexpuError of the next
:meth:`KvCache.synchronize`; torch's own synchronisation does not tell.
"""

from __future__ import annotations

import ctypes
import importlib.util

import torch

from . import LIB_DIR, PKG_DIR, TYPE_BF16, TYPE_F16, EdgexpuError, KvCacheDesc, _check, _err_buf, load_cuda

TYPES = {torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}
PAIRINGS = {"adjacent": 0, "halves": 1}


def _load():
    """The module that makes the calls (``host/kv_torch.cpp``)."""
    path = LIB_DIR / "_kv_torch.so"
    if not path.exists():
        raise ImportError(f"{path} is missing: build it with `make -C {PKG_DIR}`")
    load_cuda()
    spec = importlib.util.spec_from_file_location("_kv_torch", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.set_error(EdgexpuError)
    return module


_calls = _load()


class _Desc(KvCacheDesc):
    """The descriptor and the device of its pools, as the module reads them."""

    _fields_ = [("device", ctypes.c_int)]


class KvCache:
    """Pools k, v ``[layers][pages][kv heads][page size][head dim]`` (f16 or bf16; a page contiguous,
    layers and pages any distance apart, the same in both) and the tables over them: table int32
    ``[sequences][pages of a row]``, lens int32 ``[sequences]``, refs int32 ``[pages]``."""

    def __init__(self, k, v, table, lens, refs):
        layers, pages, n_kv, page, dim = k.shape
        if k.dtype not in (torch.float16, torch.bfloat16) or not k.is_cuda:
            raise ValueError(f"k: expected a CUDA tensor of f16 or bf16, got {k.dtype} on {k.device}")
        if v.shape != k.shape or v.dtype != k.dtype or v.stride() != k.stride() or v.device != k.device:
            raise ValueError("v must have k's shape, strides, type and device")
        if not k[0, 0].is_contiguous():
            raise ValueError("a page of k and v must be contiguous")
        layer_stride = k.stride(0) if layers > 1 else 0  # a stride that is never taken may be anything
        page_stride = k.stride(1) if pages > 1 else n_kv * page * dim
        n_seqs, columns = table.shape
        for t, shape, what in ((table, (n_seqs, columns), "table"), (lens, (n_seqs,), "lens"), (refs, (pages,), "refs")):
            if t.dtype != torch.int32 or t.device != k.device or t.shape != shape or not t.is_contiguous():
                raise ValueError(f"{what}: expected contiguous int32 of shape {shape} on {k.device}; got {t.dtype} {tuple(t.shape)} on {t.device}")
        bound = load_cuda().edgexpu_cuda_device()  # -1 before init; every call compares them again
        if bound not in (-1, k.device.index):
            raise ValueError(f"the cache is on {k.device}, the library on cuda:{bound}")
        size = load_cuda().edgexpu_cuda_kv_work_bytes(pages, n_seqs)
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self.work = torch.empty(size // 4, dtype=torch.int32, device=k.device)
        self.desc = _Desc(k.data_ptr(), v.data_ptr(), layer_stride, page_stride, TYPES[k.dtype], layers, pages,
                          page, n_kv, dim, n_seqs, columns, table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                          self.work.data_ptr(), k.device.index)
        self._desc = ctypes.addressof(self.desc)

    @classmethod
    def empty(cls, n_layers: int, n_pages: int, page_size: int, n_kv: int, head_dim: int, n_seqs: int, max_pages: int,
              dtype=torch.float16, device="cuda") -> "KvCache":
        """A cache that holds nothing."""
        k, v = (torch.empty(n_layers, n_pages, n_kv, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
        return cls(k, v, torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_seqs, dtype=torch.int32, device=device),
                   torch.zeros(n_pages, dtype=torch.int32, device=device))

    def synchronize(self) -> None:
        """Wait for torch's current stream and raise what calls of the process, this cache's among them, found wrong
        on the device since the last time."""
        buf = _err_buf()
        _check(load_cuda().edgexpu_cuda_stream_sync(torch.cuda.current_stream(self.k.device).cuda_stream, buf, 512), buf)

    # ---- pages -------------------------------------------------------------------------------------

    def append(self, seqs, n_new, missing=None):
        """Room for ``n_new[i]`` tokens more in each sequence: the first one's position, int32 (-1 where
        the pool was short, or the entry was idle).  ``missing``: int32 of one element, the pages short."""
        return _calls.append(self._desc, seqs, n_new, missing)

    def fork(self, src, dst) -> None:
        """The empty sequences ``dst`` become copies of ``src`` that share its pages."""
        _calls.fork(self._desc, src, dst)

    def free(self, seqs, keep=None) -> None:
        """Cut the sequences to their first ``keep[i]`` tokens (None: to none)."""
        _calls.free(self._desc, seqs, keep)

    def copy(self, src, dst) -> None:
        """The data of pages ``src`` into pages ``dst``, in all layers."""
        _calls.copy(self._desc, src, dst)

    def compact(self):
        """Move the pages in use to the low end of the pool; how many they are, int32 on the device."""
        return _calls.compact(self._desc)

    # ---- a layer of new tokens -----------------------------------------------------------------------

    def qk_norm_rope(self, layer: int, q, k, v, seqs, pos, n_heads: int, q_norm=None, k_norm=None, eps: float = 1e-6,
                     rope=None, pairing: str = "adjacent", out=None):
        """Norm, rotate and round the heads of new tokens; k and v into the cache, q returned as
        ``[tokens][heads][dim]`` of the cache's type.  q, k, v: fp32 ``[tokens][heads * dim]``, rows any
        distance apart.  rope: fp32 ``[positions][rotated dims]``, cos and sin of each pair."""
        return _calls.qk_norm_rope(self._desc, layer, q, k, v, seqs, pos, n_heads, q_norm, k_norm, eps, rope, PAIRINGS[pairing], out)

    def attention(self, layer: int, q, seqs, q_start=None, shared_seq: int = 0, shared_len: int = 0, max_len=None,
                  scale=None, out=None, out_dtype=None):
        """Attention of the sequences' last tokens, q ``[tokens][heads][dim]``, over the cache; the first
        ``shared_len`` positions of all sequences are those of row ``shared_seq`` and read once.  out_dtype:
        the cache's type, or float32, for which the softmax weights are kept finer (at up to a third more time)."""
        if out_dtype not in (None, self.k.dtype, torch.float32):
            raise EdgexpuError(f"attention: output type {out_dtype} (float32, or the cache's {self.k.dtype})")
        return _calls.attention(self._desc, layer, q, seqs, q_start, shared_seq, shared_len, max_len, scale, out,
                                out_dtype is torch.float32)
