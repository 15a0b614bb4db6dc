"""The decode calls' native step (csrc/b2q_host.cpp) against the binding's own
checks: the same results bit by bit, and nothing accepted that those refuse."""
import numpy as np
import pytest

import b2q
from decode_util import cuda, device, i32

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NATIVE = ("_native_plan", "_native_rope", "_native_paged", "_native_vec")


@pytest.fixture
def calls(monkeypatch):
    """[status of each native step]; plain() takes the native steps out."""
    device()
    b2q._setup()
    assert all(getattr(b2q, n) is not b2q._not_native for n in NATIVE), "the native step is not built"
    seen = []

    def watched(fn):
        def call(*args):
            seen.append(fn(*args))
            return seen[-1]
        return call
    for n in NATIVE:
        monkeypatch.setattr(b2q, n, watched(getattr(b2q, n)))

    def plain():
        for n in NATIVE:
            monkeypatch.setattr(b2q, n, b2q._not_native)
    seen_and_plain = (seen, plain)
    yield seen_and_plain


def both(calls, run):
    """run() natively and through the binding's checks: the same bits."""
    seen, plain = calls
    first = run()
    assert seen and all(s == 0 for s in seen), seen
    plain()
    for a, b in zip(first, run()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def cache(dt, n_pages=7, n_kv=2, page=4, d=16, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(n_pages, page, n_kv, d, generator=g).to(dt).cuda().transpose(1, 2)
    v = torch.randn(n_pages, page, n_kv, d, generator=g).to(dt).cuda().transpose(1, 2)
    return b2q.KVCache(k, v)


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 3])
def test_plan(calls, pad):
    def run():
        table = torch.full((3, 5 + pad), -1, dtype=torch.int32, device="cuda")
        out = [torch.full((12,), -7, dtype=torch.int32, device="cuda") for _ in range(4)]
        counts = torch.zeros(2, dtype=torch.int32, device="cuda")
        table[:, :2] = i32([9, 8, 7, 6, 5, 4]).view(3, 2)
        b2q.kv_plan(i32([5, 0, 8]), i32([1, 4, 2]), 4, i32(range(10, 16)), table[:, :5], *out, counts)
        return [table, *out, counts]
    both(calls, run)


@pytest.mark.gpu
@pytest.mark.parametrize("dt, pad, rope, norm, inter", [(F32, 0, True, True, False), (F16, 8, True, False, True),
                                                        (F16, 0, False, True, False), (F32, 8, "empty", False, False)])
def test_norm_and_rotation(calls, dt, pad, rope, norm, inter):
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(3, 6 * 16 + pad, generator=g).to(dt).cuda()[:, :96]
    table = {True: b2q.rope_table(9, 8), False: None, "empty": torch.zeros(9, 0, device="cuda")}[rope]
    w = torch.rand(16, generator=g).cuda() if norm else None

    def run():
        c, q = cache(F16), torch.zeros(3, 32 + pad, dtype=F16, device="cuda")
        b2q.qk_norm_rope(qkv, 2, c, q[:, :32], i32([0, 4, 8]), i32([3, -1, 27]), q_weight=w, k_weight=w, eps=1e-5,
                         rope=table, interleaved=inter)
        return [q, c.k.contiguous(), c.v.contiguous()]
    both(calls, run)


@pytest.mark.gpu
@pytest.mark.parametrize("dt, out, pad, seq, lse, scale", [(F16, F32, 0, False, True, None), (BF16, BF16, 8, True, False, 0.3),
                                                           (F16, F16, 8, True, True, 1)])
def test_attention(calls, dt, out, pad, seq, lse, scale):
    g = torch.Generator().manual_seed(2)
    c = cache(dt)
    q = torch.randn(3, 64 + pad, generator=g).to(dt).cuda()[:, :64]
    table = i32([0, 1, 2, 99, 3, 4, 5, 99, 6, 0, 2, 99]).view(3, 4)[:, :3]
    scratch = b2q.attention_paged_scratch(4, c)

    def run():
        o = torch.zeros(3, 64 + pad, dtype=out, device="cuda")
        e = torch.zeros(3, 4, device="cuda") if lse else None
        b2q.attention_paged(q, c, table, i32([12, 5, 0]), o[:, :64], scratch, seq_of=i32([2, 0, 1]) if seq else None,
                            scale=scale, window=7, lse=e)
        return [o] + ([e] if lse else [])
    both(calls, run)


@pytest.mark.gpu
@pytest.mark.parametrize("dt, out, pad, bias, res", [(F32, F32, 0, True, True), (F16, F16, 8, False, False),
                                                     (BF16, F32, 8, True, True)])
def test_product(calls, dt, out, pad, bias, res):
    rng = np.random.default_rng(3)
    blocks = rng.integers(0, 100, (40, 2, 18), dtype=np.uint8)
    w = b2q.WeightQ4(blocks, 40, 64)
    x = torch.from_numpy(rng.standard_normal((3, 64 + pad)).astype(np.float32)).to(dt).cuda()[:, :64]
    b = cuda(rng.standard_normal(40).astype(np.float32)) if bias else None
    r = cuda(rng.standard_normal((3, 40 + pad)).astype(np.float32))[:, :40] if res else None

    def run():
        y = torch.zeros(3, 40 + pad, dtype=out, device="cuda")
        b2q.mul_vec_q4(w, x, 3, y[:, :40], bias=b, residual=r)
        return [y]
    both(calls, run)


@pytest.mark.gpu
def test_streams(calls):
    """The current stream and a named one reach the C call."""
    w = b2q.WeightQ4(np.zeros((16, 1, 18), np.uint8), 16, 32)
    x, y = torch.ones(1, 32, device="cuda"), torch.ones(1, 16, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    before = b2q.lib().b2q_launch_count()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        b2q.mul_vec_q4(w, x, 1, y)
        b2q.mul_vec_q4(w, x, 1, y, stream=s)
    assert calls[0] == [0, 0] and b2q.lib().b2q_launch_count() == before + 2
    assert bool((y == 1).all())   # captured, not run
    g.replay()
    torch.cuda.synchronize()
    assert bool((y == 0).all())


@pytest.mark.gpu
def test_what_is_wrong_is_left_to_the_checks(calls):
    seen, _ = calls
    w = b2q.WeightQ4(np.zeros((16, 1, 18), np.uint8), 16, 32)
    x, y = torch.ones(2, 32, device="cuda"), torch.ones(2, 16, device="cuda")
    c = cache(F16)
    q, o, t, n = (torch.zeros(2, 64, dtype=F16, device="cuda"), torch.zeros(2, 64, device="cuda"),
                  i32([0, 1, 2, 3]).view(2, 2), i32([3, 4]))
    scratch = b2q.attention_paged_scratch(4, c)
    qkv, qo = torch.zeros(2, 8 * 16, device="cuda"), torch.zeros(2, 64, dtype=F16, device="cuda")
    wrong = [
        lambda: b2q.mul_vec_q4(w, x.cpu(), 2, y),
        lambda: b2q.mul_vec_q4(w, x.double(), 2, y),
        lambda: b2q.mul_vec_q4(w, x[0], 2, y),
        lambda: b2q.mul_vec_q4(w, x, 3, y),
        lambda: b2q.mul_vec_q4(w, x, 2, y[:, :15]),
        lambda: b2q.mul_vec_q4(w, x, 2, torch.ones(16, 2, device="cuda").t()),
        lambda: b2q.mul_vec_q4(w, x, 2, y, bias=torch.ones(15, device="cuda")),
        lambda: b2q.mul_vec_q4(w, x, 2, y, bias=torch.ones(16, dtype=F16, device="cuda")),
        lambda: b2q.mul_vec_q4(w, x, 2, y, residual=y.half()),
        lambda: b2q.mul_vec_q4(w, x, 2, y, residual=torch.ones(2, 20, device="cuda")[:, :16]),
        lambda: b2q.attention_paged(q.float(), c, t, n, o, scratch),
        lambda: b2q.attention_paged(q, c, t.long(), n, o, scratch),
        lambda: b2q.attention_paged(q, c, t, n.long(), o, scratch),
        lambda: b2q.attention_paged(q, c, t, n[:1], o, scratch),
        lambda: b2q.attention_paged(q, c, t, n, o[:1], scratch),
        lambda: b2q.attention_paged(q, c, t, n, o, scratch[:100]),
        lambda: b2q.attention_paged(q, c, t, n, o, scratch, seq_of=i32([0])),
        lambda: b2q.attention_paged(q, c, t, n, o, scratch, lse=torch.zeros(2, 3, device="cuda")),
        lambda: b2q.attention_paged(q[:, :60], c, t, n, o[:, :60], scratch),
        lambda: b2q.qk_norm_rope(qkv, 4, c, qo.float(), n, n),
        lambda: b2q.qk_norm_rope(qkv, 3, c, qo, n, n),
        lambda: b2q.qk_norm_rope(qkv, 4, c, qo[:1], n, n),
        lambda: b2q.qk_norm_rope(qkv, 4, c, qo, n.cpu(), n),
        lambda: b2q.qk_norm_rope(qkv, 4, c, qo, n, n[:1]),
        lambda: b2q.qk_norm_rope(qkv, 4, c, qo, n, n, q_weight=torch.ones(8, device="cuda")),
        lambda: b2q.qk_norm_rope(qkv, 4, c, qo, n, n, rope=torch.ones(8, device="cuda")),
        lambda: b2q.qk_norm_rope(qkv, 4, c, qo, n, n, rope=torch.ones(8, 8, dtype=F16, device="cuda")),
        lambda: b2q.kv_plan(n, n[:1], 4, n, t, n, n, n, n, n),
        lambda: b2q.kv_plan(n, n, 4, n, t[:1], n, n, n, n, n),
        lambda: b2q.kv_plan(n, n, 4, n.long(), t, n, n, n, n, n),
        lambda: b2q.kv_plan(n, n, 4, n, t, n, n, n, i32([1]), n),
        lambda: b2q.kv_plan(n, n, 4, n, t, n, n, n, n, i32([0, 0, 0])),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises(b2q.B2QError):
            call()
        assert seen.pop() is None and not seen, i
    # what the C entry point refuses comes back with its status
    with pytest.raises(b2q.B2QError) as e:
        b2q.kv_plan(n, n, 3, n, t, *(torch.zeros_like(n) for _ in range(5)))
    assert seen.pop() == e.value.status


def test_without_a_device_nothing_is_accepted():
    if not b2q.HOST_PATH.exists():
        pytest.skip("the native step is not built")
    b2q._setup()
    x, n = torch.ones(1, 32), torch.zeros(2, dtype=torch.int32)
    assert b2q._native_vec(1, 16, x, 1, x, None, None, None) is None
    assert b2q._native_vec(None, 16, x, 1, x, None, None, None) is None
    assert b2q._native_vec() is None
    assert b2q._native_plan(n, n, 4, n, n, n, n, n, n, n, None) is None
    assert b2q._native_rope(x, 1, None, 0, x, n, n, None, None, 1e-6, None, False, None) is None
    assert b2q._native_paged(x, None, 0, n, n, x, x, None, None, 0, None, None) is None


@pytest.mark.gpu
def test_a_cache_with_one_half_on_the_host_is_refused():
    device()
    k = torch.zeros((2, 4, 16, 64), dtype=F16, device="cuda")
    for pair in ((k, k.cpu()), (k.cpu(), k)):
        with pytest.raises(b2q.B2QError):
            b2q.KVCache(*pair)


@pytest.mark.gpu
def test_misaligned_arrays_are_refused_at_the_c_entry():
    # 32-bit entries at an odd address would fault: the call says so and launches nothing
    device()
    L, c = b2q.lib(), cache(F16)
    n = 3
    ints = [i32([0] * 16) for _ in range(9)]
    pi = [t.data_ptr() for t in ints]
    x, q = torch.zeros((n, 6 * 16), device="cuda"), torch.zeros((n, 32), dtype=F16, device="cuda")
    out, lse, w = torch.zeros((n, 32), device="cuda"), torch.zeros((n, 2), device="cuda"), torch.ones(32, device="cuda")
    rope, scratch = b2q.rope_table(4, 16), b2q.attention_paged_scratch(2, c)

    def plan(p):
        return L.b2q_kv_plan(p[0], p[1], n, 4, p[2], 4, p[3], 5, 5, n, p[4], p[5], p[6], p[7], p[8], None)

    def turn(p):
        return L.b2q_qk_norm_rope(x.data_ptr(), 0, 96, n, 2, p[0], p[1], 1e-6, p[2], 4, 16, 0, p[3], p[4],
                                  q.data_ptr(), 32, c.ref, None)

    def attend(p):
        return L.b2q_attention_paged(q.data_ptr(), 32, n, 2, c.ref, p[0], 1, 1, n, p[1], p[2], 1.0, 0, out.data_ptr(),
                                     0, 32, p[3], scratch.data_ptr(), None)

    for call, good in ((plan, pi), (turn, [w.data_ptr(), w.data_ptr(), rope.data_ptr(), pi[0], pi[1]]),
                       (attend, [pi[0], pi[1], pi[2], lse.data_ptr()])):
        before = L.b2q_launch_count()
        for i in range(len(good)):
            assert call([a + 2 * (i == j) for j, a in enumerate(good)]) == b2q.ERR_ALIGN, (call.__name__, i)
        assert L.b2q_launch_count() == before
        if call is not turn:    # (its three rows would share a slot)
            assert call(good) == b2q.OK
    torch.cuda.synchronize()
