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
_i32, _f32 = torch.int32, torch.float32
_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream() makes a Stream object: 3 us a call


def _ok(done: int) -> None:
    if not done:
        raise EdgexpuError(load_cuda().edgexpu_cuda_last_error().decode())


def _wrong(t, dtype, shape, what: str):
    return ValueError(f"{what}: expected a contiguous CUDA tensor of {dtype}, shape {tuple(shape)}; "
                      f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def _need(t, dtype, shape, what: str) -> int:
    """Address of a contiguous CUDA tensor of this type and shape."""
    if t.dtype is dtype and t.is_cuda and t.shape == shape and t.is_contiguous():
        return t.data_ptr()
    raise _wrong(t, dtype, shape, what)


def _need_rows(t, n: int, width: int, what: str) -> int:
    """Address of fp32 CUDA rows, contiguous each."""
    if t.dtype is _f32 and t.is_cuda and t.shape == (n, width) and t.stride(1) == 1:
        return t.data_ptr()
    raise ValueError(f"{what}: expected a CUDA tensor of float32, shape {(n, width)}, rows contiguous; "
                     f"got {t.dtype} {tuple(t.shape)} on {t.device}")


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
        _need(table, _i32, table.shape, "table")
        _need(lens, _i32, (n_seqs,), "lens")
        _need(refs, _i32, (pages,), "refs")
        lib = load_cuda()
        size = lib.edgexpu_cuda_kv_work_bytes(pages, n_seqs)
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self.work = torch.empty(size // 4, dtype=torch.int32, device=k.device)
        self.desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), layer_stride, page_stride, TYPES[k.dtype], layers, pages,
                                page, n_kv, dim, n_seqs, columns, table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                                self.work.data_ptr())
        self._desc = ctypes.byref(self.desc)
        self._dtype, self._device, self._index = k.dtype, k.device, k.device.index
        self._n_kv, self._dim, self._kv_width = n_kv, dim, n_kv * dim
        self._append, self._fork, self._free = lib.edgexpu_cuda_kv_append_dev, lib.edgexpu_cuda_kv_fork_dev, lib.edgexpu_cuda_kv_free_dev
        self._copy, self._compact = lib.edgexpu_cuda_kv_copy_dev, lib.edgexpu_cuda_kv_compact_dev
        self._heads, self._attend = lib.edgexpu_cuda_qk_norm_rope_dev, lib.edgexpu_cuda_kv_attention_dev
        self._attend_bytes = lib.edgexpu_cuda_kv_attention_work_bytes

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
        shape = seqs.shape
        n = shape[0]
        pos = torch.empty(n, dtype=_i32, device=self._device)
        _ok(self._append(self._desc, _need(seqs, _i32, (n,), "seqs"), _need(n_new, _i32, shape, "n_new"), n, pos.data_ptr(),
                         None if missing is None else _need(missing, _i32, (1,), "missing"), _raw_stream(self._index)))
        return pos

    def fork(self, src, dst) -> None:
        """The empty sequences ``dst`` become copies of ``src`` that share its pages."""
        n = src.shape[0]
        _ok(self._fork(self._desc, _need(src, _i32, (n,), "src"), _need(dst, _i32, (n,), "dst"), n, _raw_stream(self._index)))

    def free(self, seqs, keep=None) -> None:
        """Cut the sequences to their first ``keep[i]`` tokens (None: to none)."""
        n = seqs.shape[0]
        _ok(self._free(self._desc, _need(seqs, _i32, (n,), "seqs"), None if keep is None else _need(keep, _i32, (n,), "keep"), n,
                       _raw_stream(self._index)))

    def copy(self, src, dst) -> None:
        """The data of pages ``src`` into pages ``dst``, in all layers."""
        n = src.shape[0]
        _ok(self._copy(self._desc, _need(src, _i32, (n,), "src"), _need(dst, _i32, (n,), "dst"), n, _raw_stream(self._index)))

    def compact(self):
        """Move the pages in use to the low end of the pool; how many they are, int32 on the device."""
        live = torch.empty((), dtype=_i32, device=self._device)
        _ok(self._compact(self._desc, live.data_ptr(), _raw_stream(self._index)))
        return live

    # ---- a layer of new tokens -----------------------------------------------------------------------

    def qk_norm_rope(self, layer: int, q, k, v, seqs, pos, n_heads: int, q_norm=None, k_norm=None, eps: float = 1e-6,
                     rope=None, pairing: str = "adjacent", out=None):
        """Norm, rotate and round the heads of new tokens; k and v into the cache, q returned as
        ``[tokens][heads][dim]`` of the cache's type.  q, k, v: fp32 ``[tokens][heads * dim]``, rows any
        distance apart.  rope: fp32 ``[positions][rotated dims]``, cos and sin of each pair."""
        n, dim, wide, narrow = q.shape[0], self._dim, n_heads * self._dim, self._kv_width
        pq, pk, pv = _need_rows(q, n, wide, "q"), _need_rows(k, n, narrow, "k"), _need_rows(v, n, narrow, "v")
        if n > 1:
            wide, narrow, narrow_v = q.stride(0), k.stride(0), v.stride(0)
        else:  # the distance to a second row may be anything
            narrow_v = narrow
        if out is None:
            out = torch.empty(n, n_heads, dim, dtype=self._dtype, device=self._device)
        po = _need(out, self._dtype, (n, n_heads, dim), "out")
        pr, positions, turned = None, 0, 0
        if rope is not None:
            positions, turned = rope.shape
            pr = _need(rope, _f32, (positions, turned), "rope")
        _ok(self._heads(self._desc, layer, pq, pk, pv, wide, narrow, narrow_v, n, n_heads,
                        None if q_norm is None else _need(q_norm, _f32, (dim,), "q_norm"),
                        None if k_norm is None else _need(k_norm, _f32, (dim,), "k_norm"), eps, pr, positions, turned,
                        PAIRINGS[pairing], _need(seqs, _i32, (n,), "seqs"), _need(pos, _i32, (n,), "pos"), po,
                        _raw_stream(self._index)))
        return out

    def attention(self, layer: int, q, seqs, q_start=None, shared_seq: int = 0, shared_len: int = 0, max_len=None,
                  scale=None, out=None, out_dtype=None):
        """Attention of the sequences' last tokens, q ``[tokens][heads][dim]``, over the cache; the first
        ``shared_len`` positions of all sequences are those of row ``shared_seq`` and read once.  out_dtype:
        the cache's type, or float32."""
        tokens, heads, dim = q.shape
        batch = seqs.shape[0]
        if max_len is None:
            max_len = self.desc.max_pages * self.desc.page_size
        pq = _need(q, self._dtype, (tokens, heads, self._dim), "q")
        if out is None:
            out = torch.empty(tokens, heads, dim, dtype=out_dtype or self._dtype, device=self._device)
        po = _need(out, out.dtype, (tokens, heads, dim), "out")
        size = self._attend_bytes(self._desc, batch, tokens, heads, shared_len, max_len)
        work = torch.empty(size, dtype=torch.uint8, device=self._device) if size else None
        _ok(self._attend(self._desc, layer, pq, _need(seqs, _i32, (batch,), "seqs"),
                         None if q_start is None else _need(q_start, _i32, (batch + 1,), "q_start"), batch, tokens, heads,
                         shared_seq, shared_len, max_len, dim ** -0.5 if scale is None else scale, po,
                         TYPES.get(out.dtype, 0xFFFFFFFF), work.data_ptr() if size else None, size, _raw_stream(self._index)))
        return out
