"""A batch served over the paged cache: prompts, parallel samples, penalties, a grammar.

    python -m aero_b200.serve_example [--steps 32] [--temperature 0.8 --top-p 0.9] [--blocks 4]

A small decoder with random weights (embedding, per layer grouped-query attention over
`PagedCache` and the MoE block of `CudaMoeLayer`, a head) serves three prompts: one
call takes all prompt tokens, every prompt is forked into parallel samples, each
decode step takes one token of every sample and adjusts its logits (`logits.adjust`:
penalties from its history, a bias against the end token, a mask of allowed tokens)
before the next one is drawn (`logits.sample`: the largest, unless a temperature is given). Samples
that end are freed and the pool is compacted. Odd layers attend within a window, with the first tokens kept
visible; with `blocks`, decode steps of the even layers attend to that many blocks that `select` chooses.
"""

from __future__ import annotations

import argparse
import math


class PagedDecoder:
    """The decoder: random weights of a seed, f16 activations in attention, f32 elsewhere."""

    def __init__(self, cache, n_head: int, d: int, vocab: int, window: int = 0, sinks: int = 0, seed: int = 0,
                 blocks: int = 0) -> None:
        import torch
        from . import synth
        from .quant import DTYPE_Q8_0
        self.torch, self.cache, self.H, self.d, self.vocab = torch, cache, n_head, d, vocab
        self.window, self.sinks, self.blocks = window, sinks, blocks
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def w(rows, cols):
            return torch.randn((rows, cols), device="cuda", generator=g).mul_(1 / math.sqrt(cols))

        D, HK = cache.head_dim, cache.n_head_kv
        self.embed, self.head = w(vocab, d).mul_(math.sqrt(d)), w(vocab, d)
        self.layers = [(w((n_head + 2 * HK) * D, d), w(d, n_head * D)) for _ in range(cache.n_layer)]
        self.moe = [synth.open_layer(synth.make_layer(synth.LayerSpec(d, 16, 4, 256, 0, DTYPE_Q8_0), seed + i))
                    for i in range(cache.n_layer)]
        # one stream for the MoE handles, torch and the cache (which follows torch's current stream)
        self.stream = torch.cuda.Stream()
        for m in self.moe:
            m.set_stream(self.stream)
        # rotary angles of half the head
        self.freq = 1e4 ** (-torch.arange(D // 2, device="cuda") / (D // 2))
        self.stream.wait_stream(torch.cuda.current_stream())  # the weights above are made on the caller's stream

    def _norm(self, x):
        return x * self.torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)

    def _rotate(self, x, positions):
        a = positions[:, None, None] * self.freq
        x0, x1 = x.chunk(2, -1)
        return self.torch.cat([x0 * a.cos() - x1 * a.sin(), x0 * a.sin() + x1 * a.cos()], -1)

    def forward(self, tokens, row_seq, positions, seqs, q_start=None):
        """Logits of the last token of each of seqs. tokens, row_seq, positions: one entry a
        token, its sequence and position, whose room was taken with cache.extend; q_start as for
        attend. All int32 CUDA tensors; call within `self.stream`."""
        torch, c = self.torch, self.cache
        D, HK, T = c.head_dim, c.n_head_kv, tokens.numel()
        x = self.embed[tokens.long()]
        for i, (qkv, o) in enumerate(self.layers):
            y = (self._norm(x) @ qkv.T).view(T, self.H + 2 * HK, D)
            q, k = self._rotate(self._norm(y[:, :self.H]), positions), self._rotate(self._norm(y[:, self.H:-HK]), positions)
            c.append(i, k.to(c.dtype), y[:, -HK:].to(c.dtype), row_seq, positions)
            q = q.to(c.dtype)
            if self.blocks and q_start is None and i % 2 == 0:
                a = c.attend_blocks(i, q, seqs, c.select(i, q, seqs, n_blocks=self.blocks))
            else:
                a = c.attend(i, q, seqs, q_start, window=self.window if i % 2 else 0, sinks=self.sinks)
            x = x + a.reshape(T, -1).float() @ o.T
            x = x + self.moe[i].forward(self._norm(x))
        last = x if q_start is None else x[(q_start[1:] - 1).long()]
        return self._norm(last) @ self.head.T

    def close(self) -> None:
        self.torch.cuda.synchronize()
        for m in self.moe:
            m.close()


def i32(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def mask_of(allowed, vocab: int, rows: int):
    """Packed bits of the allowed token ids, the same for every row."""
    import numpy as np
    import torch
    bits = np.zeros((vocab + 31) // 32 * 32, np.uint8)
    bits[allowed] = 1
    words = np.packbits(bits, bitorder="little").view(np.int32)
    return torch.from_numpy(words).cuda().expand(rows, -1).contiguous()


def serve(steps: int = 32, samples: int = 2, seed: int = 0, d: int = 256, vocab: int = 1000, layers: int = 2,
          temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, blocks: int = 0) -> dict:
    """Serves three prompts with `samples` samples each; returns their tokens and the cache's state. The largest
    logit is taken, or with a temperature a token is drawn; blocks: see the top."""
    import torch
    from .logits import adjust, sample
    from .pages import PagedCache
    prompts = [[(7 * i + j * j) % vocab for j in range(n)] for i, n in enumerate((5, 70, 33))]
    P, n_seq, end = 16, len(prompts) * (samples + 1), vocab - 1
    longest = max(map(len, prompts)) + steps
    cache = PagedCache(layers, n_seq * (longest // P + 2), P, 2, 64, n_seq, longest // P + 2, dtype=torch.float16,
                       bounds=blocks > 0)
    net = PagedDecoder(cache, 8, d, vocab, window=32, sinks=4, seed=seed, blocks=blocks)
    numbers = torch.Generator(device="cuda").manual_seed(seed)  # the random numbers that tokens are drawn with
    with torch.cuda.stream(net.stream):
        # all prompts in one call
        roots = list(range(len(prompts)))
        start = [0]
        for p in prompts:
            start.append(start[-1] + len(p))
        cache.extend(i32(roots), i32([len(p) for p in prompts]))
        flat = i32([t for p in prompts for t in p])
        first = net.forward(flat, i32([s for s, p in enumerate(prompts) for _ in p]),
                            i32([j for p in prompts for j in range(len(p))]), i32(roots), i32(start))
        # each prompt continued several ways: sample k begins with the prompt's k-th best token
        live = [len(prompts) + s * samples + k for s in roots for k in range(samples)]
        cache.fork(i32([s for s in roots for _ in range(samples)]), i32(live))
        cache.free(i32(roots))
        best = first.topk(samples, dim=1).indices
        history = torch.zeros((n_seq, longest + 1), dtype=torch.int32, device="cuda")
        n = [0] * n_seq
        for s in roots:
            for k in range(samples):
                row = len(prompts) + s * samples + k
                history[row, :len(prompts[s])] = flat[start[s]:start[s + 1]]
                history[row, len(prompts[s])] = best[s, k].int()
                n[row] = len(prompts[s]) + 1
        n_prompt = [0] * len(prompts) + [len(prompts[s]) for s in roots for _ in range(samples)]
        allowed = [t for t in range(vocab) if t % 3 or t == end]  # the "grammar"
        compacted = 0
        for step in range(steps - 1):
            B = len(live)
            seqs, rows = i32(live), torch.tensor(live, device="cuda")
            held = i32([n[s] for s in live])
            cache.extend(seqs, i32([1] * B))
            tok = history[rows, (held - 1).long()]
            logits = net.forward(tok, seqs, held - 1, seqs)
            adjust(logits, history=history[rows], n_history=held, n_prompt=i32([n_prompt[s] for s in live]),
                   repetition=torch.full((B,), 1.2, device="cuda"), frequency=torch.full((B,), 0.1, device="cuda"),
                   presence=torch.full((B,), 0.2, device="cuda"), bias_start=i32(list(range(B + 1))),
                   bias_token=i32([end] * B), bias_value=torch.full((B,), -1.0, device="cuda"),
                   mask=mask_of(allowed, vocab, B), out=logits)
            nxt = sample(logits, torch.rand(B, device="cuda", generator=numbers), temperature=torch.full((B,), temperature, device="cuda"),
                         top_k=i32([top_k] * B), top_p=torch.full((B,), top_p, device="cuda"),
                         min_p=torch.full((B,), min_p, device="cuda"))
            history[rows, held.long()] = nxt
            for s in live:
                n[s] += 1
            # the first sample of the second prompt stops half-way, as one that met its end token would
            ended = [s for s, t in zip(live, nxt.tolist()) if t == end or (step == steps // 2 and s == len(prompts) + samples)]
            if ended:
                cache.free(i32(ended))
                cache.compact()
                compacted += 1
                live = [s for s in live if s not in ended]
            if not live:
                break
        cache.check()
        table, length, refs = (x.clone() for x in cache.tables())
        out = {"prompts": prompts, "history": history.cpu(), "n": n, "live": live, "length": length.cpu(),
               "pages": int((refs > 0).sum()), "highest": int(refs.nonzero().max()) if live else -1, "compacted": compacted,
               "allowed": allowed, "samples": samples}
    net.close()
    cache.close()
    return out


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=32)
    p.add_argument("--samples", type=int, default=2)
    p.add_argument("--temperature", type=float, default=0.0, help="0: the largest logit")
    p.add_argument("--top-k", type=int, default=0)
    p.add_argument("--top-p", type=float, default=1.0)
    p.add_argument("--min-p", type=float, default=0.0)
    p.add_argument("--blocks", type=int, default=0, help="blocks that a decode step's even layers attend to; 0: all")
    a = p.parse_args()
    r = serve(a.steps, a.samples, temperature=a.temperature, top_k=a.top_k, top_p=a.top_p, min_p=a.min_p, blocks=a.blocks)
    for row, n in enumerate(r["n"]):
        if n:
            print(f"sequence {row}: {r['history'][row, :n].tolist()}")
    print(f"{len(r['live'])} sequences live in {r['pages']} pages (highest number {r['highest']}), {r['compacted']} compactions")


if __name__ == "__main__":
    main()
