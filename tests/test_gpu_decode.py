"""The decode operators together, as b2q.decode runs them, against the decoder in
64 bits over each request's whole sequence.

Tolerance, from the arithmetic: keys, values and queries are rounded to 11 bits,
and the two feed-forward products of a layer quantize their inputs to 1/127 of a
block's largest value, which is about three times its rms: an error of half a step
is 3 / 254 / sqrt(3) = 0.7% of a product's result.  With two layers the logits, which
the residual stream dominates, are off by less than 2% of their norm, their
direction by 1 - 0.02^2 / 2.
"""
import numpy as np
import pytest

import b2q
from b2q import synth
from b2q.decode import Decoder, DecoderConfig
from decode_util import device

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

CFG = DecoderConfig(hidden=256, ffn=500, n_head=4, n_kv_head=2, n_layer=2, vocab=501, max_pos=256)


@pytest.fixture(scope="module", autouse=True)
def dev():
    device()


class Weights:
    """Quantized weights for the decoder, and the same values in 64 bits."""

    def __init__(self, cfg, seed=0):
        rng = np.random.default_rng(seed)
        self.cfg, self.layers, self.exact = cfg, [], []

        def normal(*shape, std=0.05):
            return (std * rng.standard_normal(shape)).astype(np.float32)

        def q4(n, k):
            q = synth.quantize_q4_0(normal(n, k))
            return b2q.WeightQ4(q, n, k), synth.dequantize_q4_0(q, k).astype(np.float64)

        def q8(n, k):
            kp = -(-k // 32) * 32
            q = synth.quantize_q8_0(normal(n, k), kp)
            return b2q.Weight(q, n, kp), synth.dequantize_q8_0(q, kp).astype(np.float64)[:, :k]

        for _ in range(cfg.n_layer):
            mats = dict(qkv=q4(cfg.qkv, cfg.hidden), out=q4(cfg.hidden, cfg.hidden), fc1=q8(cfg.ffn, cfg.hidden),
                        fc2=q8(cfg.hidden, cfg.ffn))
            vecs = dict(qkv_b=normal(cfg.qkv), out_b=normal(cfg.hidden), fc1_b=normal(cfg.ffn), fc2_b=normal(cfg.hidden),
                        ln1_w=1 + normal(cfg.hidden), ln1_b=normal(cfg.hidden), ln2_w=1 + normal(cfg.hidden),
                        ln2_b=normal(cfg.hidden), q_norm=1 + normal(cfg.d_head), k_norm=1 + normal(cfg.d_head))
            self.layers.append({**{k: v[0] for k, v in mats.items()},
                                **{k: torch.from_numpy(v).cuda() for k, v in vecs.items()}})
            self.exact.append({**{k: v[1] for k, v in mats.items()},
                               **{k: v.astype(np.float64) for k, v in vecs.items()}})
        self.head, self.head_exact = q4(cfg.vocab, cfg.hidden)
        self.final = (1 + normal(cfg.hidden), normal(cfg.hidden))

    def decoder(self, **kw):
        return Decoder(self.cfg, self.layers, self.head, *(torch.from_numpy(v).cuda() for v in self.final), **kw)

    def logits(self, x):
        """After the last of x [n][hidden]."""
        c, n = self.cfg, x.shape[0]
        d, half = c.d_head, c.d_head // 2
        ang = np.arange(n)[:, None] * 10000.0 ** (-2.0 * np.arange(half) / d)

        def ln(v, w, b):
            m = v.mean(1, keepdims=True)
            return (v - m) / np.sqrt(((v - m) ** 2).mean(1, keepdims=True) + c.eps) * w + b

        def turn(h, w):
            h = h / np.sqrt((h * h).mean(-1, keepdims=True) + c.eps) * w
            a, b, cos, sin = h[..., :half], h[..., half:], np.cos(ang)[:, None], np.sin(ang)[:, None]
            return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)

        x = x.astype(np.float64)
        for w in self.exact:
            y = (ln(x, w["ln1_w"], w["ln1_b"]) @ w["qkv"].T + w["qkv_b"]).reshape(n, -1, d)
            q = turn(y[:, :c.n_head], w["q_norm"])
            k = turn(y[:, c.n_head:c.n_head + c.n_kv_head], w["k_norm"]).repeat(c.n_head // c.n_kv_head, 1)
            v = y[:, c.n_head + c.n_kv_head:].repeat(c.n_head // c.n_kv_head, 1)
            s = np.einsum("ihd,jhd->hij", q, k) / np.sqrt(d)
            s = np.where(np.tril(np.ones((n, n), bool)), s, -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))
            o = np.einsum("hij,jhd->ihd", p / p.sum(-1, keepdims=True), v).reshape(n, -1)
            x = x + o @ w["out"].T + w["out_b"]
            z = ln(x, w["ln2_w"], w["ln2_b"]) @ w["fc1"].T + w["fc1_b"]
            z = 0.5 * z * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
            x = x + z @ w["fc2"].T + w["fc2_b"]
        return ln(x[-1:], *(v.astype(np.float64) for v in self.final))[0] @ self.head_exact.T


def run(dec, seqs, new, rows, rng):
    """One step in which request s brings new[s] random embeddings; seqs is extended."""
    parts = [rng.standard_normal((n, CFG.hidden)).astype(np.float32) for n in new]
    for s, p in enumerate(parts):
        seqs[s] = np.concatenate([seqs[s], p])
    flat = np.concatenate(parts)
    dec.x[:len(flat)] = torch.from_numpy(flat).cuda()
    dec.new_len.copy_(torch.tensor(new, dtype=torch.int32))
    return dec.step(rows)


def check(w, logits, seqs, new):
    got = logits.double().cpu().numpy()
    for s, n in enumerate(new):
        if n:
            ref = w.logits(seqs[s])
            err = np.linalg.norm(got[s] - ref) / np.linalg.norm(ref)
            cos = got[s] @ ref / np.linalg.norm(got[s]) / np.linalg.norm(ref)
            assert err <= 0.02 and cos >= 1 - 2e-4, (s, err, cos)


def test_prompts_and_steps_of_ragged_requests():
    w, rng = Weights(CFG), np.random.default_rng(5)
    dec = w.decoder(max_requests=3, max_rows=64, n_pages=40)
    seqs = [np.zeros((0, CFG.hidden), np.float32) for _ in range(3)]
    # an image's prefix first, then others join; padding rows behind the tokens
    for new, rows in [([40, 0, 0], 40), ([1, 17, 0], 20), ([1, 1, 5], 64), ([1, 0, 1], 2), ([1, 1, 1], 3),
                      ([0, 16, 30], 50)]:
        check(w, run(dec, seqs, new, rows, rng), seqs, new)
        assert b2q.check_device() == 0
    assert dec.ctx_len.tolist() == [len(s) for s in seqs]
    owned = [p for r in dec.table.tolist() for p in r if p >= 0]
    free = [p for p in dec.free.tolist() if p >= 0]
    assert sorted(owned + free) == list(range(40))
    # a request ends and another takes its place, on its pages
    dec.release(1)
    seqs[1] = seqs[1][:0]
    check(w, run(dec, seqs, [1, 33, 1], 35, rng), seqs, [1, 33, 1])
    assert b2q.check_device() == 0


def test_running_out_of_pages_is_reported():
    w, rng = Weights(CFG), np.random.default_rng(6)
    dec = w.decoder(max_requests=2, max_rows=64, n_pages=3)
    seqs = [np.zeros((0, CFG.hidden), np.float32) for _ in range(2)]
    check(w, run(dec, seqs, [20, 10], 30, rng), seqs, [20, 10])
    assert b2q.check_device() == 0
    run(dec, seqs, [15, 1], 16, rng)
    with pytest.raises(b2q.B2QError):
        b2q.check_device()


def test_captured_steps_replay_while_the_lengths_grow():
    w, rng = Weights(CFG), np.random.default_rng(7)
    eager, graphed = (w.decoder(max_requests=3, max_rows=32, n_pages=40) for _ in range(2))
    for d in (eager, graphed):
        run(d, [np.zeros((0, CFG.hidden), np.float32) for _ in range(3)], [3, 14, 15], 32, np.random.default_rng(8))
    rows = torch.from_numpy(rng.standard_normal((8, 3, CFG.hidden)).astype(np.float32)).cuda()
    for d in (eager, graphed):
        d.new_len.fill_(1)
    x = torch.empty((3, CFG.hidden), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x.copy_(rows[0])
    with torch.cuda.stream(side):
        graphed.x[:3] = x
        graphed.step(3)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.x[:3] = x
        graphed.step(3)
    eager.x[:3] = rows[0]
    eager.step(3)
    for i in range(1, 8):
        x.copy_(rows[i])
        graph.replay()
        eager.x[:3] = rows[i]
        assert torch.equal(eager.step(3), graphed.logits)
    assert torch.equal(eager.ctx_len, graphed.ctx_len) and b2q.check_device() == 0


def test_a_request_alone_and_in_company():
    w, rng = Weights(CFG), np.random.default_rng(9)
    one, many = w.decoder(max_requests=1, max_rows=32, n_pages=20), w.decoder(max_requests=5, max_rows=64, n_pages=60)
    mine = rng.standard_normal((21, CFG.hidden)).astype(np.float32)
    one.x[:21] = torch.from_numpy(mine).cuda()
    one.new_len.fill_(21)
    a = one.step(21)[0].double()
    new = [3, 21, 9, 1, 7]
    flat = rng.standard_normal((sum(new), CFG.hidden)).astype(np.float32)
    flat[3:24] = mine
    many.x[:len(flat)] = torch.from_numpy(flat).cuda()
    many.new_len.copy_(torch.tensor(new, dtype=torch.int32))
    b = many.step(len(flat))[1].double()
    # the same arithmetic in another order: what the roundings to 16 and 8 bits make of that
    assert ((a - b).norm() / a.norm()).item() <= 0.02


def test_more_requests_than_rows_of_a_step():
    # the last LayerNorm has a row per request: its activations need room for them
    w, rng = Weights(CFG), np.random.default_rng(10)
    dec = w.decoder(max_requests=70, max_rows=5, n_pages=40)
    assert dec.act_h.numel() >= b2q.act_empty(70, CFG.hidden).numel()
    seqs = [np.zeros((0, CFG.hidden), np.float32) for _ in range(70)]
    for busy in ({3: 4, 69: 1}, {69: 5}, {0: 1, 3: 1, 40: 2, 69: 1}):
        new = [busy.get(s, 0) for s in range(70)]
        check(w, run(dec, seqs, new, 5, rng), seqs, new)
        assert b2q.check_device() == 0


def pages_of(dec):
    """Every page that a request owns (up to its length) or that is free."""
    owned = [p for r, n in zip(dec.table.tolist(), dec.ctx_len.tolist()) for p in r[:-(-n // dec.page_size)]]
    assert min(owned, default=0) >= 0
    free = dec.free.tolist()
    left = [p for p in free if p >= 0]
    assert free[:len(left)] == left             # no hole
    return sorted(owned + left)


def test_tokens_without_a_row_are_reported_and_not_counted():
    w, rng = Weights(CFG), np.random.default_rng(11)
    dec = w.decoder(max_requests=4, max_rows=20, n_pages=40)
    seqs = [np.zeros((0, CFG.hidden), np.float32) for _ in range(4)]
    check(w, run(dec, seqs, [6, 0, 3, 0], 9, rng), seqs, [6, 0, 3, 0])
    # 54 tokens, 20 rows: 15 of the first request's, 5 of the second's, none of the others
    flat = rng.standard_normal((20, CFG.hidden)).astype(np.float32)
    dec.x[:] = torch.from_numpy(flat).cuda()
    dec.new_len.copy_(torch.tensor([15, 35, 4, 0], dtype=torch.int32))
    logits = dec.step(20)
    with pytest.raises(b2q.B2QError) as e:
        b2q.check_device()
    assert "code 8" in str(e.value)
    seqs[0], seqs[1] = np.concatenate([seqs[0], flat[:15]]), flat[15:]
    check(w, logits, seqs, [1, 1, 1, 0])        # (the third one's last token is still its last)
    assert dec.ctx_len.tolist() == [21, 5, 3, 0] and pages_of(dec) == list(range(40))
    check(w, run(dec, seqs, [1, 14, 2, 3], 20, rng), seqs, [1, 14, 2, 3])
    assert b2q.check_device() == 0 and pages_of(dec) == list(range(40))


def test_tokens_without_a_page_or_a_position_are_not_counted():
    w, rng = Weights(CFG), np.random.default_rng(12)
    dec = w.decoder(max_requests=2, max_rows=64, n_pages=3)
    seqs = [np.zeros((0, CFG.hidden), np.float32) for _ in range(2)]
    check(w, run(dec, seqs, [20, 10], 30, rng), seqs, [20, 10])
    run(dec, seqs, [15, 1], 16, rng)
    with pytest.raises(b2q.B2QError):
        b2q.check_device()
    assert dec.ctx_len.tolist() == [32, 11] and pages_of(dec) == [0, 1, 2]
    seqs[0] = seqs[0][:32]
    check(w, run(dec, seqs, [0, 5], 5, rng), seqs, [0, 5])
    assert b2q.check_device() == 0 and dec.ctx_len.tolist() == [32, 16]
    # the block table ends at position 256, before the pages do
    dec = w.decoder(max_requests=1, max_rows=64, n_pages=40)
    seqs = [np.zeros((0, CFG.hidden), np.float32)]
    for _ in range(4):
        run(dec, seqs, [63], 63, rng)
    assert b2q.check_device() == 0
    run(dec, seqs, [9], 9, rng)
    with pytest.raises(b2q.B2QError):
        b2q.check_device()
    assert dec.ctx_len.tolist() == [256] and pages_of(dec) == list(range(40))


def test_pages_after_they_ran_out():
    # run out, release, go on, release twice: every page is owned or free, exactly once
    w, rng = Weights(CFG), np.random.default_rng(13)
    dec = w.decoder(max_requests=3, max_rows=64, n_pages=6)
    seqs = [np.zeros((0, CFG.hidden), np.float32) for _ in range(3)]

    def out_of_pages(new):
        run(dec, seqs, new, sum(new), rng)
        with pytest.raises(b2q.B2QError):
            b2q.check_device()
        for s in range(3):
            seqs[s] = seqs[s][:int(dec.ctx_len[s])]
        assert pages_of(dec) == list(range(6))

    def release(s):
        dec.release(s)
        seqs[s] = seqs[s][:0]
        assert pages_of(dec) == list(range(6))

    check(w, run(dec, seqs, [20, 10, 30], 60, rng), seqs, [20, 10, 30])
    out_of_pages([31, 15, 10])
    assert dec.ctx_len.tolist() == [48, 16, 32]
    release(1)
    check(w, run(dec, seqs, [10, 0, 0], 10, rng), seqs, [10, 0, 0])
    out_of_pages([10, 3, 0])
    assert dec.ctx_len.tolist() == [64, 0, 32]
    release(0)
    release(2)
    check(w, run(dec, seqs, [20, 30, 14], 64, rng), seqs, [20, 30, 14])
    assert b2q.check_device() == 0 and pages_of(dec) == list(range(6))


def test_requests_that_have_brought_nothing_have_the_logits_of_zeros():
    w, rng = Weights(CFG), np.random.default_rng(14)
    taken = [torch.full((3, CFG.hidden), float("nan"), device="cuda") for _ in range(64)]
    del taken                                   # memory that the decoder's buffers may get
    dec = w.decoder(max_requests=3, max_rows=8, n_pages=8)
    logits = run(dec, [np.zeros((0, CFG.hidden), np.float32)] * 3, [0, 4, 0], 4, rng).double().cpu().numpy()
    ref = w.final[1].astype(np.float64) @ w.head_exact.T     # the last LayerNorm of zeros is its bias
    for s in (0, 2):
        assert np.linalg.norm(logits[s] - ref) <= 1e-5 * np.linalg.norm(ref)
