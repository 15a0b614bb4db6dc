"""Answering with tokens: a small decoder on the library's kernels.

The towers encode; this runs what follows them, a decoder of the towers' block
shape (pre-LN, GELU feed-forward, optionally fewer key heads) over a paged
key-value cache.  A step takes any mix of requests: one new token each, whole
prompts (rows of the hidden width: token embeddings, or features of the caller's;
the towers give one pooled vector an image and no patch features), idle ones.  Per step

  kv_plan              block tables, positions and slots from the lengths

and per layer

  ln_quantize          LayerNorm (its fp32 output feeds the 4-bit product)
  mul_vec_q4           [Q | K | V] = x W + b                    (Q4_0 / Q4_1)
  qk_norm_rope         norm and rotation, keys and values to the cache
  attention_paged      over each request's pages
  mul_vec_q4           output projection + bias + residual
  ln_quantize, mul_mat feed-forward with Q8_0 weights (GELU -> q8_1, residual)

and logits of each request's last row from a 4-bit head.  Every computation is a
library call; torch holds the memory and looks up token embeddings.  A step
on the same number of rows launches the same kernels on the same buffers, so it
can be captured in a CUDA graph once and replayed while the lengths grow.

    python -m b2q.decode        (in hbd-siglip2.cpp_b200/: steps/s on random weights)
"""
from __future__ import annotations

from dataclasses import dataclass

import b2q


@dataclass
class DecoderConfig:
    hidden: int = 1152
    ffn: int = 4304
    n_head: int = 16
    n_kv_head: int = 16
    n_layer: int = 27
    vocab: int = 256000
    max_pos: int = 4096
    eps: float = 1e-6

    @property
    def d_head(self) -> int:
        return self.hidden // self.n_head

    @property
    def qkv(self) -> int:
        return (self.n_head + 2 * self.n_kv_head) * self.d_head


def placed_tokens(seq_of, slot, new_len):
    """What a plan (its seq_of and slot of a step's rows) has done for each request:
    how many of its new tokens have a row and a cache slot, and the row of the last of
    them.  Rows and pages run out from the end, so these are the first of the tokens
    that the request brings."""
    import torch
    count = torch.zeros_like(new_len).index_add_(0, seq_of.clamp(min=0), (slot >= 0).to(torch.int32))
    new = new_len.clamp(min=0)
    return count, (torch.cumsum(new, 0) - new + count - 1).clamp(0, seq_of.numel() - 1)


def entered_pages(slot, page_size: int):
    """How many pages these rows are the first ones of: those of a plan that hold a token."""
    return ((slot & (page_size - 1 - 2 ** 31)) == 0).sum()     # (the sign too: -1 is no slot)


class Decoder:
    """layers: a list of dicts with "qkv", "out" (b2q.WeightQ4), "fc1", "fc2"
    (b2q.Weight), their fp32 biases "qkv_b", "out_b", "fc1_b", "fc2_b", fp32
    "ln1_w", "ln1_b", "ln2_w", "ln2_b" [hidden] and "q_norm", "k_norm" [d_head];
    head: WeightQ4 [vocab][hidden]; final_w, final_b: the last LayerNorm."""

    def __init__(self, cfg: DecoderConfig, layers, head, final_w, final_b, max_requests: int, max_rows: int,
                 n_pages: int, page_size: int = 16):
        import torch
        self.cfg, self.layers, self.head, self.final = cfg, layers, head, (final_w, final_b)
        self.max_rows, self.page_size = max_rows, page_size
        dev, h, r = "cuda", cfg.hidden, max_rows

        def f32(*shape):
            return torch.empty(shape, dtype=torch.float32, device=dev)

        def i32(*shape):
            return torch.zeros(shape, dtype=torch.int32, device=dev)

        self.caches = [b2q.KVCache(*(torch.zeros((n_pages, cfg.n_kv_head, page_size, cfg.d_head), dtype=torch.float16,
                                                 device=dev) for _ in range(2))) for _ in layers]
        width = -(-cfg.max_pos // page_size)
        self.rope = b2q.rope_table(width * page_size, cfg.d_head)   # every position that the table has a page for
        self.ctx_len, self.new_len = i32(max_requests), i32(max_requests)
        self.table = torch.full((max_requests, width), -1, dtype=torch.int32, device=dev)
        self.free = torch.arange(n_pages, dtype=torch.int32, device=dev)
        self._iota = torch.arange(n_pages, device=dev)
        self.seq_of, self.pos, self.slot, self.kv_len, self.counts = i32(r), i32(r), i32(r), i32(r), i32(2)
        self.x, self.y, self.qkv, self.attn = f32(r, h), f32(r, h), f32(r, cfg.qkv), f32(r, h)
        self.q = torch.empty((r, h), dtype=torch.float16, device=dev)
        # the layers' rows, and at the end one row per request
        self.act_h, self.act_f = b2q.act_empty(max(r, max_requests), h), b2q.act_empty(r, cfg.ffn)
        # a request that has brought nothing yet has a last row of zeros
        self.last, self.logits = f32(max_requests, h).zero_(), f32(max_requests, cfg.vocab)
        self.last_n = f32(max_requests, h)
        self.scratch = b2q.attention_paged_scratch(cfg.n_head, self.caches[0])

    def step(self, rows: int):
        """One step over `rows` rows: self.x[:rows] holds the new tokens'
        embeddings, requests in order, self.new_len how many each request brings
        (their sum at most rows; rows beyond it are padding).  Returns the
        logits [requests][vocab] after each request's last new token (rows of
        idle requests are those of whatever they had last), valid until the
        next step.  B2QError where rows is not in 1..max_rows.

        Tokens that get no row, page or position are left out and reported by
        b2q.check_device: self.ctx_len grows by what was cached, no page is taken for
        the others, and logits are those after the last token that was."""
        import torch
        if not 1 <= rows <= self.max_rows:
            raise b2q.B2QError(b2q.ERR_SHAPE, f"a step takes 1 to {self.max_rows} rows, not {rows}")
        c, r = self.cfg, rows
        x, y, qkv, q, attn = self.x[:r], self.y[:r], self.qkv[:r], self.q[:r], self.attn[:r]
        seq_of, pos, slot, kv_len = self.seq_of[:r], self.pos[:r], self.slot[:r], self.kv_len[:r]
        b2q.kv_plan(self.ctx_len, self.new_len, self.page_size, self.free, self.table, seq_of, pos, slot, kv_len,
                    self.counts)
        placed, at = placed_tokens(seq_of, slot, self.new_len)
        # the list moves up by the pages that hold a token, -1 behind its last; those
        # planned for tokens without a row are the last ones and stay in it (their table
        # entries are behind the request's length: the next plan enters them anew)
        after = self._iota + entered_pages(slot, self.page_size)
        self.free.copy_(torch.where(after < after.numel(), self.free[after.clamp(max=after.numel() - 1)], -1))
        for w, cache in zip(self.layers, self.caches):
            b2q.ln_quantize(x, w["ln1_w"], w["ln1_b"], c.eps, r, c.hidden, self.act_h, y)
            b2q.mul_vec_q4(w["qkv"], y, r, qkv, bias=w["qkv_b"])
            b2q.qk_norm_rope(qkv, c.n_head, cache, q, pos, slot, w["q_norm"], w["k_norm"], c.eps, self.rope)
            b2q.attention_paged(q, cache, self.table, kv_len, attn, self.scratch, seq_of=seq_of)
            b2q.mul_vec_q4(w["out"], attn, r, x, bias=w["out_b"], residual=x)
            b2q.ln_quantize(x, w["ln2_w"], w["ln2_b"], c.eps, r, c.hidden, self.act_h)
            b2q.mul_mat(w["fc1"], self.act_h, r, kind=b2q.EPI_BIAS_GELU_Q8, bias=w["fc1_b"], act_out=self.act_f)
            b2q.mul_mat(w["fc2"], self.act_f, r, x, kind=b2q.EPI_BIAS_RESIDUAL, bias=w["fc2_b"], residual=x)
        self.ctx_len += placed
        n = self.ctx_len.numel()
        self.last.copy_(torch.where((placed > 0)[:, None], x[at], self.last))
        b2q.ln_quantize(self.last, *self.final, c.eps, n, c.hidden, self.act_h, self.last_n)
        b2q.mul_vec_q4(self.head, self.last_n, n, self.logits)
        return self.logits

    def release(self, request: int):
        """Ends a request: its pages are free again (synchronises)."""
        row = self.table[request, :-(-int(self.ctx_len[request]) // self.page_size)]
        pages, left = row[row >= 0], int((self.free >= 0).sum())
        self.free[left:left + pages.numel()] = pages
        self.ctx_len[request] = 0
        self.table[request] = -1


def random_decoder(cfg: DecoderConfig, seed: int = 0, std: float = 0.02, **kw) -> Decoder:
    """A decoder with seeded N(0, std) weights quantized as a checkpoint's would be."""
    import numpy as np
    import torch

    from . import synth
    rng = np.random.default_rng(seed)

    def normal(*shape):
        return (std * rng.standard_normal(shape)).astype(np.float32)

    def q4(n, k):
        return b2q.WeightQ4(synth.quantize_q4_0(normal(n, k)), n, k)

    def q8(n, k):
        kp = -(-k // 32) * 32
        return b2q.Weight(synth.quantize_q8_0(normal(n, k), kp), n, kp)

    def dev(a):
        return torch.from_numpy(a).cuda()

    layers = []
    for _ in range(cfg.n_layer):
        layers.append(dict(
            qkv=q4(cfg.qkv, cfg.hidden), out=q4(cfg.hidden, cfg.hidden), fc1=q8(cfg.ffn, cfg.hidden),
            fc2=q8(cfg.hidden, cfg.ffn), qkv_b=dev(normal(cfg.qkv)), out_b=dev(normal(cfg.hidden)),
            fc1_b=dev(normal(cfg.ffn)), fc2_b=dev(normal(cfg.hidden)), ln1_w=dev(1 + normal(cfg.hidden)),
            ln1_b=dev(normal(cfg.hidden)), ln2_w=dev(1 + normal(cfg.hidden)), ln2_b=dev(normal(cfg.hidden)),
            q_norm=dev(1 + normal(cfg.d_head)), k_norm=dev(1 + normal(cfg.d_head))))
    return Decoder(cfg, layers, q4(cfg.vocab, cfg.hidden), dev(1 + normal(cfg.hidden)), dev(normal(cfg.hidden)), **kw)


def main():
    import argparse

    import torch
    p = argparse.ArgumentParser(description="decode steps per second on random weights (one CUDA graph per step)")
    p.add_argument("--requests", type=int, default=4)
    p.add_argument("--context", type=int, default=729, help="cached tokens per request at the start")
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--layers", type=int, default=27)
    p.add_argument("--vocab", type=int, default=32000)
    a = p.parse_args()
    b2q.init(0)
    cfg = DecoderConfig(n_layer=a.layers, vocab=a.vocab)
    pages = a.requests * (-(-(a.context + a.steps + 8) // 16) + 1)
    d = random_decoder(cfg, max_requests=a.requests, max_rows=a.requests, n_pages=pages)
    g = torch.Generator(device="cuda").manual_seed(0)
    for c in d.caches:   # a prefix of a.context tokens, as if it had been prefilled
        c.k.normal_(generator=g)
        c.v.normal_(generator=g)
    have = -(-a.context // d.page_size)
    d.table[:, :have] = d.free[:a.requests * have].view(a.requests, have)
    d.free.copy_(torch.roll(d.free, -a.requests * have))
    d.free[d.free.numel() - a.requests * have:] = -1
    d.ctx_len.fill_(a.context)
    d.new_len.fill_(1)
    embed = 0.02 * torch.randn(cfg.vocab, cfg.hidden, device="cuda", generator=g)
    ids = torch.zeros(a.requests, dtype=torch.int64, device="cuda")

    def step():
        d.x[:a.requests] = embed[ids]
        ids.copy_(d.step(a.requests).argmax(1))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(a.steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    b2q.check_device()
    ms = begin.elapsed_time(end) / a.steps
    print(f"{a.layers} layers, {a.requests} requests from {a.context} tokens: {ms:.3f} ms a step, "
          f"{1e3 * a.requests / ms:.0f} tokens/s")


if __name__ == "__main__":
    main()
