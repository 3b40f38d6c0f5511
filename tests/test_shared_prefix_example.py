"""The batch of requests behind one prompt (examples/shared_prefix_batch.py): the paged cache, the norm +
rotation + store and the shared-prefix attention between the library's linears, end to end."""

import importlib.util

import numpy as np
import pytest

from _oracle import REPO

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("shared_prefix_batch", REPO / "examples" / "shared_prefix_batch.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def float_linears(gpu, example):
    """The example's decoder with its weights dequantized: the library's linears quantize their input rows,
    and a rounding of the attention's can move such a quant by a whole step."""

    class Decoder(example.Decoder):
        def _linear(self, x, weight, n_out):
            w = torch.empty(n_out, x.shape[1], device="cuda")
            self._ok(self.cuda.edgexpu_cuda_dequantize_rows_dev(w.data_ptr(), weight, self.type, None, n_out, x.shape[1],
                                                                torch.cuda.current_stream().cuda_stream))
            return x @ w.T

        def _linears(self, x, weights, n_outs):
            return [self._linear(x, w, n) for w, n in zip(weights, n_outs)]

    return Decoder(gpu)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_hidden_states_with_and_without_sharing_and_of_one_request_alone(gpu, example, dtype):
    """A decode step of five requests: the prefix read once for all, read by each, and one request alone in
    another cache give the same hidden rows but for the attention's rounding of its weights and inputs, a few
    2^-11 (f16) or 2^-8 (bf16) of the rows' size (two layers, each adding at most a few of those)."""
    from edgexpu_llm_b200.kv import KvCache

    model = float_linears(gpu, example)
    try:
        rng = np.random.default_rng(5)
        prompt = rng.integers(0, model.vocab, 333).tolist()
        questions = [rng.integers(0, model.vocab, n).tolist() for n in (1, 7, 30, 2, 16)]
        rows = {}
        for share in (True, False):
            cache = KvCache.empty(model.layers, 80, 16, model.n_kv, model.dim, 6, 40, dtype=dtype)
            example.generate(model, cache, prompt, questions, 1, share)
            ids = example.ints([11, 12, 13, 14, 15])
            seqs = example.ints([1, 2, 3, 4, 5])
            pos = cache.append(seqs, example.ints([1] * 5))
            assert pos.tolist() == [333 + len(q) for q in questions]
            rows[share] = model.hidden(cache, ids, seqs, pos, seqs, None, 333 if share else 0)
        cache = KvCache.empty(model.layers, 80, 16, model.n_kv, model.dim, 2, 40, dtype=dtype)
        alone = prompt + questions[2] + [13]
        cache.append(example.ints([1]), example.ints([len(alone)]))
        n = len(alone)
        single = model.hidden(cache, example.ints(alone), example.ints([1] * n), torch.arange(n, dtype=torch.int32, device="cuda"),
                              example.ints([1]), example.ints([0, n]), 0)[-1]
        unit = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
        size = rows[True].norm(dim=1)
        assert bool(((rows[True] - rows[False]).norm(dim=1) <= 16 * unit * size).all())
        assert float((rows[True][2] - single).norm()) <= 16 * unit * float(size[2])
    finally:
        model.close()


def test_generation_frees_and_packs_its_pages(gpu, example):
    from edgexpu_llm_b200.kv import KvCache

    model = example.Decoder(gpu, layers=1)
    try:
        cache = KvCache.empty(1, 60, 16, model.n_kv, model.dim, 5, 30)
        out = example.generate(model, cache, list(range(50)), [[1, 2, 3], [4], [5, 6], [7]], 12)
        assert out.shape == (4, 12) and bool(((out >= 0) & (out < model.vocab)).all())
        assert cache.lens.tolist() == [50, 64, 62, 63, 62]
        held = 4 + 4  # the prompt's pages, and each request's copy of its partly filled last one
        assert int((cache.refs > 0).sum()) == held
        cache.free(example.ints([1, 3]))
        assert int(cache.compact()) == held - 2
        assert int(cache.table.max()) == held - 3
        cache.free(example.ints([0, 2, 4]))
        assert not cache.refs.any() and not cache.lens.any() and int(cache.table.max()) == -1
    finally:
        model.close()
