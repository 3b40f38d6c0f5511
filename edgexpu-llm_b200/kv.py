"""A key/value cache in pages that many sequences share, on torch tensors.

:class:`KvCache` binds the ``edgexpu_cuda_kv_*`` and ``edgexpu_cuda_qk_norm_rope_dev`` calls of
``include/edgexpu_cuda.h``, which say what each call does.  Tensors live on the library's device and
calls run on torch's current stream; none of them waits for the device.
"""

from __future__ import annotations

import ctypes

import torch

from . import TYPE_BF16, TYPE_F16, TYPE_F32, EdgexpuError, KvCacheDesc, load_cuda

TYPES = {torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16, torch.float32: TYPE_F32}
PAIRINGS = {"adjacent": 0, "halves": 1}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ok(done: int) -> None:
    if not done:
        raise EdgexpuError(load_cuda().edgexpu_cuda_last_error().decode())


def _need(t, dtype, shape, what: str):
    """Address of a contiguous CUDA tensor of this type and shape (None in `shape`: any extent)."""
    if t.dtype != dtype or not t.is_cuda or not t.is_contiguous() or len(t.shape) != len(shape) or any(
            b is not None and a != b for a, b in zip(t.shape, shape)):
        raise ValueError(f"{what}: expected a contiguous CUDA tensor of {dtype}, shape {tuple(shape)}; "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


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
        _need(table, torch.int32, (None, None), "table")
        _need(lens, torch.int32, (n_seqs,), "lens")
        _need(refs, torch.int32, (pages,), "refs")
        self._lib = load_cuda()
        size = self._lib.edgexpu_cuda_kv_work_bytes(pages, n_seqs)
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self.work = torch.empty(size // 4, dtype=torch.int32, device=k.device)
        self.desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), layer_stride, page_stride, TYPES[k.dtype], layers, pages,
                                page, n_kv, dim, n_seqs, columns, table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                                self.work.data_ptr())
        self._desc = ctypes.byref(self.desc)

    @classmethod
    def empty(cls, n_layers: int, n_pages: int, page_size: int, n_kv: int, head_dim: int, n_seqs: int, max_pages: int,
              dtype=torch.float16, device="cuda") -> "KvCache":
        """A cache that holds nothing."""
        k, v = (torch.empty(n_layers, n_pages, n_kv, page_size, head_dim, dtype=dtype, device=device) for _ in range(2))
        return cls(k, v, torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_seqs, dtype=torch.int32, device=device),
                   torch.zeros(n_pages, dtype=torch.int32, device=device))

    # ---- pages -------------------------------------------------------------------------------------

    def append(self, seqs, n_new, missing=None):
        """Room for ``n_new[i]`` tokens more in each sequence: the first one's position, int32 (-1 where
        the pool was short, or the entry was idle).  ``missing``: int32 of one element, the pages short."""
        n = seqs.shape[0]
        pos = torch.empty(n, dtype=torch.int32, device=self.table.device)
        _ok(self._lib.edgexpu_cuda_kv_append_dev(
            self._desc, _need(seqs, torch.int32, (n,), "seqs"), _need(n_new, torch.int32, (n,), "n_new"), n, pos.data_ptr(),
            None if missing is None else missing.data_ptr(), _stream()))
        return pos

    def fork(self, src, dst) -> None:
        """The empty sequences ``dst`` become copies of ``src`` that share its pages."""
        n = src.shape[0]
        _ok(self._lib.edgexpu_cuda_kv_fork_dev(self._desc, _need(src, torch.int32, (n,), "src"),
                                               _need(dst, torch.int32, (n,), "dst"), n, _stream()))

    def free(self, seqs, keep=None) -> None:
        """Cut the sequences to their first ``keep[i]`` tokens (None: to none)."""
        n = seqs.shape[0]
        _ok(self._lib.edgexpu_cuda_kv_free_dev(self._desc, _need(seqs, torch.int32, (n,), "seqs"),
                                               None if keep is None else _need(keep, torch.int32, (n,), "keep"), n, _stream()))

    def copy(self, src, dst) -> None:
        """The data of pages ``src`` into pages ``dst``, in all layers."""
        n = src.shape[0]
        _ok(self._lib.edgexpu_cuda_kv_copy_dev(self._desc, _need(src, torch.int32, (n,), "src"),
                                               _need(dst, torch.int32, (n,), "dst"), n, _stream()))

    def compact(self):
        """Move the pages in use to the low end of the pool; how many they are, int32 on the device."""
        live = torch.empty((), dtype=torch.int32, device=self.table.device)
        _ok(self._lib.edgexpu_cuda_kv_compact_dev(self._desc, live.data_ptr(), _stream()))
        return live

    # ---- a layer of new tokens -----------------------------------------------------------------------

    def qk_norm_rope(self, layer: int, q, k, v, seqs, pos, n_heads: int, q_norm=None, k_norm=None, eps: float = 1e-6,
                     rope=None, pairing: str = "adjacent", out=None):
        """Norm, rotate and round the heads of new tokens; k and v into the cache, q returned as
        ``[tokens][heads][dim]`` of the cache's type.  q, k, v: fp32 ``[tokens][heads * dim]``, rows any
        distance apart.  rope: fp32 ``[positions][rotated dims]``, cos and sin of each pair."""
        d = self.desc
        n = q.shape[0]
        for t, heads, what in ((q, n_heads, "q"), (k, d.n_kv, "k"), (v, d.n_kv, "v")):
            if t.dtype != torch.float32 or not t.is_cuda or t.shape != (n, heads * d.head_dim) or t.stride(1) != 1:
                raise ValueError(f"{what}: expected a CUDA tensor of float32, shape {(n, heads * d.head_dim)}; "
                                 f"got {t.dtype} {tuple(t.shape)}")
        if out is None:
            out = torch.empty(n, n_heads, d.head_dim, dtype=self.k.dtype, device=self.k.device)
        weights = [None if w is None else _need(w, torch.float32, (d.head_dim,), "norm weight") for w in (q_norm, k_norm)]
        table = (None, 0, 0) if rope is None else (_need(rope, torch.float32, (None, None), "rope"), *rope.shape)
        _ok(self._lib.edgexpu_cuda_qk_norm_rope_dev(
            self._desc, layer, q.data_ptr(), k.data_ptr(), v.data_ptr(), *(t.stride(0) if n > 1 else t.shape[1] for t in (q, k, v)), n, n_heads,
            *weights, eps, *table, PAIRINGS[pairing], _need(seqs, torch.int32, (n,), "seqs"),
            _need(pos, torch.int32, (n,), "pos"), _need(out, self.k.dtype, (n, n_heads, d.head_dim), "out"), _stream()))
        return out

    def attention(self, layer: int, q, seqs, q_start=None, shared_seq: int = 0, shared_len: int = 0, max_len=None,
                  scale=None, out=None, out_dtype=None):
        """Attention of the sequences' last tokens, q ``[tokens][heads][dim]``, over the cache; the first
        ``shared_len`` positions of all sequences are those of row ``shared_seq`` and read once.  out_dtype:
        the cache's type, or float32."""
        d = self.desc
        tokens, heads, batch = q.shape[0], q.shape[1], seqs.shape[0]
        max_len = d.max_pages * d.page_size if max_len is None else max_len
        if out is None:
            out = torch.empty(q.shape, dtype=out_dtype or q.dtype, device=q.device)
        size = self._lib.edgexpu_cuda_kv_attention_work_bytes(self._desc, batch, tokens, heads, shared_len, max_len)
        work = torch.empty(size, dtype=torch.uint8, device=q.device)
        _ok(self._lib.edgexpu_cuda_kv_attention_dev(
            self._desc, layer, _need(q, self.k.dtype, (tokens, heads, d.head_dim), "q"), _need(seqs, torch.int32, (batch,), "seqs"),
            None if q_start is None else _need(q_start, torch.int32, (batch + 1,), "q_start"), batch, tokens, heads, shared_seq,
            shared_len, max_len, d.head_dim ** -0.5 if scale is None else scale,
            _need(out, out.dtype, q.shape, "out"), TYPES.get(out.dtype, 0xFFFFFFFF), work.data_ptr(), size, _stream()))
        return out
