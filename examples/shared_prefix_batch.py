"""Several requests behind one prompt: the paged cache and its attention beside the library's linears.

A llama-shaped decoder of random Q8_0 weights reads a prompt once, forks it into requests of their own
(no data moves), gives each its question, and decodes them together, greedily:

    append   room for the new tokens (the forks' last page becomes their own)
    layer    RMSNorm, q|k|v in one launch, norm + rotation + store, attention behind the shared prefix
             (fp32 out, the next linear's input), o, RMSNorm, gate|up in one launch, SwiGLU, down
    logits   greedy argmax over the logits weight, a row at a time
    free     a request's pages go back when it is done; compact packs what is left

Run it on a B200:  python examples/shared_prefix_batch.py [requests] [new tokens]
(With random weights the best ids are close calls, which a rounding can decide otherwise.)
"""

from __future__ import annotations

import ctypes
import importlib.util
import pathlib
import sys
import time

import numpy as np
import torch

ROOT = pathlib.Path(__file__).resolve().parent.parent


def load_package():
    name = "edgexpu_llm_b200"
    if name not in sys.modules:
        path = ROOT / "edgexpu-llm_b200"
        spec = importlib.util.spec_from_file_location(name, path / "__init__.py", submodule_search_locations=[str(path)])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


class Decoder:
    """A decoder of `layers` llama layers with normed query and key heads; weights uploaded once."""

    def __init__(self, pkg, layers=2, n_embd=576, heads=9, n_kv=3, n_ff=1536, vocab=4096, positions=4096, seed=0):
        from edgexpu_llm_b200 import synth

        self.pkg, self.cuda, self.type = pkg, pkg.load_cuda(), pkg.TYPE_Q8_0
        self.layers, self.n_embd, self.heads, self.n_kv, self.n_ff, self.vocab = layers, n_embd, heads, n_kv, n_ff, vocab
        self.dim = n_embd // heads
        rng = np.random.default_rng(seed)

        def weight(n_out, n_in):
            return pkg.upload_weight(synth.weight(rng, self.type, n_out, n_in), self.type, n_out, n_in)

        kv = n_kv * self.dim
        self.embd, self.logits = weight(vocab, n_embd), weight(vocab, n_embd)
        self.w = [{"q": weight(n_embd, n_embd), "k": weight(kv, n_embd), "v": weight(kv, n_embd), "o": weight(n_embd, n_embd),
                   "gate": weight(n_ff, n_embd), "up": weight(n_ff, n_embd), "down": weight(n_embd, n_ff)} for _ in range(layers)]
        gen = torch.Generator().manual_seed(seed)
        self.head_norms = [[(1 + 0.1 * torch.randn(self.dim, generator=gen)).cuda() for _ in range(2)] for _ in range(layers)]
        freq = 10000.0 ** (-torch.arange(0, self.dim, 2, dtype=torch.float64) / self.dim)
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
        self.rope = torch.stack([angle.cos(), angle.sin()], -1).reshape(positions, self.dim).float().cuda()

    def close(self):
        for h in [self.embd, self.logits] + [h for layer in self.w for h in layer.values()]:
            self.pkg.free_weight(h)

    def _ok(self, done):
        if not done:
            raise self.pkg.EdgexpuError(self.cuda.edgexpu_cuda_last_error().decode())

    def _linear(self, x, weight, n_out):
        out = torch.empty(x.shape[0], n_out, device=x.device)
        self._ok(self.cuda.edgexpu_cuda_linear_quant_batch_dev(out.data_ptr(), x.data_ptr(), weight, self.type, None, x.shape[0], n_out,
                                                               x.shape[1], torch.cuda.current_stream().cuda_stream))
        return out

    def _linears(self, x, weights, n_outs):
        """Linears that read the same rows, in one launch."""
        outs = [torch.empty(x.shape[0], n, device=x.device) for n in n_outs]
        self._ok(self.cuda.edgexpu_cuda_linear_quant_multi_dev(
            len(outs), (ctypes.c_void_p * len(outs))(*(o.data_ptr() for o in outs)), (ctypes.c_void_p * len(outs))(*weights),
            (ctypes.c_int * len(outs))(*n_outs), None, self.type, x.data_ptr(), x.shape[0], x.shape[1],
            torch.cuda.current_stream().cuda_stream))
        return outs

    @staticmethod
    def _norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def hidden(self, cache, ids, seqs, pos, rows, starts, shared_len):
        """The last hidden rows of the tokens `ids` (int32), token t being position pos[t] of sequence seqs[t];
        rows and starts say which tokens are whose (starts None: one token each)."""
        n, stream = ids.shape[0], torch.cuda.current_stream().cuda_stream
        x = torch.empty(n, self.n_embd, device="cuda")
        self._ok(self.cuda.edgexpu_cuda_dequantize_rows_dev(x.data_ptr(), self.embd, self.type, ids.data_ptr(), n, self.n_embd, stream))
        kv = self.n_kv * self.dim
        for i, w in enumerate(self.w):
            q, k, v = self._linears(self._norm(x), [w["q"], w["k"], w["v"]], [self.n_embd, kv, kv])
            q_norm, k_norm = self.head_norms[i]
            q = cache.qk_norm_rope(i, q, k, v, seqs, pos, n_heads=self.heads, q_norm=q_norm, k_norm=k_norm, rope=self.rope)
            a = cache.attention(i, q, rows, q_start=starts, shared_seq=0, shared_len=shared_len, out_dtype=torch.float32)
            x = x + self._linear(a.reshape(n, self.n_embd), w["o"], self.n_embd)
            gate, up = self._linears(self._norm(x), [w["gate"], w["up"]], [self.n_ff, self.n_ff])
            x = x + self._linear(torch.nn.functional.silu(gate) * up, w["down"], self.n_embd)
        return self._norm(x)

    def greedy(self, hidden):
        """The best id of each row, int32 on the device."""
        keys = torch.zeros(hidden.shape[0], dtype=torch.int64, device="cuda")
        for i in range(hidden.shape[0]):
            self._ok(self.cuda.edgexpu_cuda_logits_argmax_dev(self.logits, self.type, hidden[i].data_ptr(), self.n_embd, self.vocab, None, 0,
                                                              keys[i:].data_ptr(), torch.cuda.current_stream().cuda_stream))
        return (0xFFFFFFFF - (keys & 0xFFFFFFFF)).int()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def generate(model, cache, prompt, questions, new_tokens, share=True):
    """Greedy continuations of prompt + question, [request][new token]; row 0 of the cache keeps the prompt.
    share: whether attention reads the prompt once for all."""
    n = len(questions)
    rows = ints(list(range(1, n + 1)))
    at = cache.append(ints([0]), ints([len(prompt)]))
    pos = at + torch.arange(len(prompt), dtype=torch.int32, device="cuda")
    model.hidden(cache, ints(prompt), ints([0] * len(prompt)), pos, ints([0]), ints([0, len(prompt)]), 0)
    cache.fork(ints([0] * n), rows)

    counts = [len(q) for q in questions]
    starts = [sum(counts[:i]) for i in range(n + 1)]
    owner = torch.repeat_interleave(torch.arange(n, device="cuda"), ints(counts).long())
    at = cache.append(rows, ints(counts))
    pos = (at[owner] + torch.arange(starts[-1], device="cuda") - ints(starts)[owner]).int()
    shared_len = len(prompt) if share else 0
    hidden = model.hidden(cache, ints([t for q in questions for t in q]), rows[owner].contiguous(), pos, rows, ints(starts), shared_len)
    ids = model.greedy(hidden[ints(starts)[1:].long() - 1].contiguous())
    out, one = [ids], ints([1] * n)
    for _ in range(new_tokens - 1):
        pos = cache.append(rows, one)
        ids = model.greedy(model.hidden(cache, ids, rows, pos, rows, None, shared_len))
        out.append(ids)
    return torch.stack(out, 1)


def main():
    requests = int(sys.argv[1]) if len(sys.argv) > 1 else 16
    new_tokens = int(sys.argv[2]) if len(sys.argv) > 2 else 32
    pkg = load_package()
    pkg.init(0)
    from edgexpu_llm_b200.kv import KvCache

    model = Decoder(pkg)
    rng = np.random.default_rng(1)
    prompt = rng.integers(0, model.vocab, 1000).tolist()
    questions = [rng.integers(0, model.vocab, rng.integers(1, 20)).tolist() for _ in range(requests)]
    for share in (False, True, False, True):
        cache = KvCache.empty(model.layers, 64 + 8 * requests, 16, model.n_kv, model.dim, requests + 1, 128)
        torch.cuda.synchronize()
        t = time.perf_counter()
        out = generate(model, cache, prompt, questions, new_tokens, share)
        cache.synchronize()  # and what the calls found wrong on the device
        print(f"prompt {'read once for all' if share else 'read by each'}: {time.perf_counter() - t:.3f} s, "
              f"first ids {out[0, :6].tolist()}, pages in use {int((cache.refs > 0).sum())}")
        cache.free(ints(list(range(1, requests // 2 + 1))))
        print(f"  half of the requests given back, pages in use after packing: {int(cache.compact())}")
        cache.synchronize()
    model.close()
    pkg.shutdown()


if __name__ == "__main__":
    main()
