"""Search, then answer: the encoder finds chunks of code, and a decoder reads them once and writes several
answers over that shared context.

The chunks are embedded and searched with ``EmbedBackend`` and ``SearchIndex``.  The tokens of the best chunks
become a prefix, whose keys and values are computed once (one causal prompt) and then shared by every answer
of the batch: ``DecodeStep`` plans each step, ``append`` rotates the queries and keys and writes the cache,
``attend`` reads the prefix and each answer's own keys, ``rms_norm`` is the decoder's norm.  The weights are
random (there are none to load here), so the answers mean nothing; the program shows the calls and times them.

    python examples/answer_over_context.py [--answers 16] [--tokens 32]
"""

from __future__ import annotations

import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from ripvec_b200 import EmbedBackend, ModelSpec, synth  # noqa: E402
from ripvec_b200.decode import DecodeStep, PagedCache, rms_norm  # noqa: E402
from ripvec_b200.index import SearchIndex  # noqa: E402


@dataclass(frozen=True)
class DecoderSpec:
    hidden: int = 512
    layers: int = 2
    q_heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    intermediate: int = 1024
    vocab: int = 1000
    max_position: int = 4096
    page_size: int = 32
    pages: int = 512
    rope_theta: float = 10000.0
    eps: float = 1e-5


class Decoder:
    """A pre-norm decoder over a paged cache; one instance holds one cache."""

    def __init__(self, spec: DecoderSpec, seed: int = 0, dtype=torch.bfloat16, device: int = 0):
        s, dev = spec, torch.device("cuda", device)
        g = torch.Generator(device=dev).manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=dev) * shape[-1] ** -0.5).to(dtype)

        self.spec, self.device, self.dtype = s, dev, dtype
        rows = (s.q_heads + 2 * s.kv_heads) * s.head_dim
        self.embedding = torch.randn(s.vocab, s.hidden, generator=g, device=dev).to(dtype)
        self.layers = [dict(qkv=w(rows, s.hidden), o=w(s.hidden, s.q_heads * s.head_dim),
                            up=w(2 * s.intermediate, s.hidden), down=w(s.hidden, s.intermediate),
                            norm1=torch.ones(s.hidden, device=dev), norm2=torch.ones(s.hidden, device=dev))
                       for _ in range(s.layers)]
        self.norm = torch.ones(s.hidden, device=dev)
        inv = s.rope_theta ** (-torch.arange(0, s.head_dim, 2, device=dev) / s.head_dim)
        angle = torch.arange(s.max_position, device=dev)[:, None] * inv
        self.cos, self.sin = angle.cos(), angle.sin()
        pool = (s.layers, 2, s.pages, s.kv_heads, s.page_size, s.head_dim)
        self.pool = torch.empty(pool, dtype=dtype, device=dev)
        self.caches = [PagedCache(p[0], p[1]) for p in self.pool]
        self.step = DecodeStep(q_heads=s.q_heads, kv_heads=s.kv_heads, head_dim=s.head_dim, page_size=s.page_size,
                               device=device)
        self.free = list(range(s.pages))

    def take_pages(self, tokens: int) -> list[int]:
        """Pages for `tokens` more keys of a sequence that starts on a new page."""
        need = -(-tokens // self.spec.page_size)
        if need > len(self.free):
            raise RuntimeError("the cache is full")
        taken, self.free = self.free[:need], self.free[need:]
        return taken

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        """Logits of the planned step's new tokens (``ids``, packed)."""
        s, t = self.spec, ids.shape[0]
        residual, x = self.embedding[ids], None
        for layer, cache in zip(self.layers, self.caches):
            if x is None:
                h, _ = rms_norm(residual, layer["norm1"], eps=s.eps)
            else:
                h, _ = rms_norm(x, layer["norm1"], residual=residual, residual_out=residual, eps=s.eps)
            qkv = (h @ layer["qkv"].T).view(t, -1, s.head_dim)
            q, k, v = qkv.split((s.q_heads, s.kv_heads, s.kv_heads), dim=1)
            q = self.step.append(cache, q, k, v, self.cos, self.sin)
            x = self.step.attend(cache, q).view(t, -1) @ layer["o"].T
            h, _ = rms_norm(x, layer["norm2"], residual=residual, residual_out=residual, eps=s.eps)
            gate, up = (h @ layer["up"].T).chunk(2, dim=-1)
            x = (torch.nn.functional.silu(gate) * up) @ layer["down"].T
        h, _ = rms_norm(x, self.norm, residual=residual, eps=s.eps)
        return h @ self.embedding.T

    def read(self, ids: torch.Tensor) -> dict:
        """Computes the keys and values of a context once; returns its pages and length."""
        n = ids.shape[0]
        pages = self.take_pages(n)
        self.step.plan(q_lens=[n], own_lens=[n], own_pages=[pages], num_pages=self.spec.pages)
        self.forward(ids)
        return dict(pages=pages, length=n)

    def answer(self, context: dict, prompts: list[torch.Tensor], tokens: int) -> torch.Tensor:
        """Greedy answers of `tokens` tokens to each prompt over one shared context: ``[prompts, tokens]``."""
        lens = [len(p) for p in prompts]
        pages = [self.take_pages(n + tokens) for n in lens]
        new, ids, out = lens, torch.cat(prompts), []
        own = [0] * len(prompts)
        for _ in range(tokens):
            own = [a + b for a, b in zip(own, new)]
            self.step.plan(q_lens=new, own_lens=own, own_pages=pages, prefix_lens=[context["length"]],
                           prefix_pages=[context["pages"]], num_pages=self.spec.pages)
            last = torch.tensor(new, device=self.device).cumsum(0) - 1
            ids = self.forward(ids)[last].argmax(-1)
            out.append(ids)
            new = [1] * len(prompts)
        for p in pages:
            self.free += p
        return torch.stack(out, 1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--answers", type=int, default=16)
    ap.add_argument("--tokens", type=int, default=32)
    a = ap.parse_args()
    spec = ModelSpec("modernbert", 256, 2, 4, 256, 1000, 512)
    backend = EmbedBackend(spec, synth.random_weights(spec, seed=1))
    chunks, cu = synth.packed_ids(synth.uniform_lengths(200, 64, 400, seed=2), spec.vocab, seed=3)
    index = SearchIndex(backend.embed_packed(chunks, cu))
    question, qcu = synth.packed_ids(synth.uniform_lengths(1, 12, 12, seed=4), spec.vocab, seed=5)
    best = index.topk(backend.embed_packed(question, qcu), 3)[0][0]
    context = torch.cat([torch.from_numpy(chunks[cu[i]:cu[i + 1]]).long() for i in best]).cuda()

    decoder = Decoder(DecoderSpec())
    read = decoder.read(context)
    prompts = [torch.from_numpy(question).long().cuda()] * a.answers
    decoder.answer(read, prompts, 2)  # warm-up
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    out = decoder.answer(read, prompts, a.tokens)
    end.record()
    torch.cuda.synchronize()
    print(f"chunks {best.tolist()}: {len(context)} tokens read once; {a.answers} answers of {a.tokens} tokens in "
          f"{begin.elapsed_time(end):.1f} ms; first answer {out[0, :8].tolist()} ...")


if __name__ == "__main__":
    main()
