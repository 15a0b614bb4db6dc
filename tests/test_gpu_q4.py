"""b2q_mul_vec_q4 against the product in 64 bits, and the block formats against
gguf-py's decoder.

Tolerance, from the arithmetic: products and sums in fp32 over blocks of 32 and
then over the blocks, so at most 32 + K/32 + 8 roundings of 2^-23 of the sum of
absolute terms (|d q x| and |m x| apart); one rounding to the output's type.
"""
import numpy as np
import pytest

import b2q
from decode_util import TINY, UNIT, device, within

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
Q4_0, Q4_1 = b2q.GGML_Q4_0, b2q.GGML_Q4_1


@pytest.fixture(scope="module", autouse=True)
def dev():
    device()


def blocks(rng, n, k, typ):
    """Random blocks: (bytes [n][k/32][18 or 20], weights and their terms' sizes in 64 bits)."""
    b = rng.integers(0, 256, (n, k // 32, 18 if typ == Q4_0 else 20), dtype=np.uint8)
    d = (0.01 * rng.standard_normal((n, k // 32, 1))).astype(np.float16)
    b[..., :2] = d.view(np.uint8)
    q = b[..., 2:] if typ == Q4_0 else b[..., 4:]
    q = np.concatenate([q & 15, q >> 4], -1).astype(np.float64)
    if typ == Q4_0:
        w = (q - 8) * d
        return b, w.reshape(n, k), np.abs(w).reshape(n, k)
    m = (0.05 * rng.standard_normal((n, k // 32, 1))).astype(np.float16)
    b[..., 2:4] = m.view(np.uint8)
    return b, (q * d + m).reshape(n, k), (np.abs(q * d) + np.abs(m)).reshape(n, k)


def check(m, n, k, typ=Q4_0, dt=F32, out=None, bias=False, res=False, x_cols=None, ldx=0, ldy=0, in_place=False,
          host=False, row_pad=0, offset=0, scale=1.0, stream=None):
    rng = np.random.default_rng(m * 7919 + n * 31 + k)
    out = out or dt
    b, w, mag = blocks(rng, n, k, typ)
    cols = x_cols or k
    x = (scale * rng.standard_normal((m, cols + ldx))).astype(np.float32)
    flat = torch.zeros(m * (cols + ldx) + offset, dtype=dt, device="cuda")
    flat[offset:] = torch.from_numpy(x).to(dt).reshape(-1).cuda()
    xd = flat[offset:].view(m, cols + ldx)[:, :cols]
    if ldx:   # what lies between the rows is not read
        flat[offset:].view(m, cols + ldx)[:, cols:] = float("nan")
    raw = np.full((n, b[0].size + row_pad), 255, np.uint8)
    raw[:, :b[0].size] = b.reshape(n, -1)
    W = b2q.WeightQ4(raw if host else torch.from_numpy(raw).cuda(), n, k, typ, row_bytes=raw.shape[1])
    bt = torch.from_numpy(rng.standard_normal(n).astype(np.float32)).cuda() if bias else None
    y = torch.full((m, n + ldy), 5.0, dtype=out, device="cuda")
    rt = None
    if res:
        rt = torch.from_numpy(rng.standard_normal((m, n + ldy)).astype(np.float32)).cuda()
        if in_place:
            y.copy_(rt)
    before = None if rt is None else rt.double().cpu().numpy()[:, :n]
    keep = y[:, n:].clone()
    torch.cuda.synchronize()
    b2q.mul_vec_q4(W, xd, m, y[:, :n], bt, y[:, :n] if in_place else (None if rt is None else rt[:, :n]),
                   stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(y[:, n:], keep)
    x64 = xd.double().cpu().numpy()
    ref = x64 @ w[:, :cols].T
    tol = (32 + k / 32 + 8) * 2.0 ** -23 * (np.abs(x64) @ mag[:, :cols].T)
    for extra in ([bt.double().cpu().numpy()[None]] if bias else []) + ([before] if res else []):
        ref = ref + extra
        tol = tol + 2.0 ** -23 * (np.abs(ref) + np.abs(extra))
    within(y[:, :n].double().cpu().numpy(), ref, tol + UNIT[out] * 1.01 * np.abs(ref) + TINY[out])
    W.release()


@pytest.mark.parametrize("typ", [Q4_0, Q4_1], ids=["q4_0", "q4_1"])
@pytest.mark.parametrize("dt, out", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("m", [1, 2, 3, 8, 9])
def test_types_and_rows(typ, dt, out, m):
    check(m, 200, 256, typ, dt, out)


@pytest.mark.parametrize("n, k", [(1, 32), (1, 96), (15, 32), (16, 64), (17, 2048), (129, 4320), (1152, 1152), (8, 20000),
                                  (40000, 64)])
@pytest.mark.parametrize("typ", [Q4_0, Q4_1], ids=["q4_0", "q4_1"])
def test_sizes(typ, n, k):
    check(1, n, k, typ)
    check(3, n, k, typ, BF16)


@pytest.mark.parametrize("m", [1, 5, 16, 33, 70])
def test_more_rows_than_a_pass(m):
    check(m, 333, 1152, Q4_1, F32)
    check(m, 333, 1152, Q4_0, F16)


def test_long_columns_for_several_rows():
    check(8, 100, 14336, Q4_0, F32)
    check(6, 100, 28672, Q4_1, F16, F32)


@pytest.mark.parametrize("cols", [4289, 4304, 4319])
def test_columns_short_of_a_block(cols):
    check(1, 70, 4320, Q4_0, F32, x_cols=cols)
    check(2, 70, 4320, Q4_1, BF16, F32, x_cols=cols)


def test_epilogue():
    check(1, 300, 320, bias=True)
    check(3, 300, 320, res=True)
    check(3, 300, 320, bias=True, res=True, in_place=True, ldy=5)
    check(3, 300, 320, Q4_1, F16, F16, bias=True, res=True)


def test_strides_and_alignment():
    check(4, 100, 256, ldx=3, ldy=1)
    check(4, 100, 256, Q4_1, F16, ldx=5, offset=1)
    check(1, 100, 256, Q4_0, BF16, offset=3)
    check(2, 100, 256, Q4_1, F32, row_pad=7, host=True)
    check(2, 100, 256, Q4_0, F32, row_pad=7)


@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1e4, 1e30])
def test_activation_ranges(scale):
    # fp32 activations keep their 24 bits and their range
    check(2, 100, 512, Q4_0, F32, scale=scale)
    check(2, 100, 512, Q4_1, F32, scale=scale)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("head, tail", [(0.0, 1.0), (1e-3, 50.0), (1.0, 3e4), (100.0, 1e-2)])
def test_rows_whose_first_columns_say_nothing_of_the_rest(dt, head, tail):
    # the operands' scale is guessed from a row's first 32 values: zeros, far smaller or far larger ones
    rng = np.random.default_rng(11)
    b, w, mag = blocks(rng, 100, 1024, Q4_0)
    x = rng.standard_normal((3, 1024)).astype(np.float32)
    x[:, :32] *= head
    x[:, 32:] *= 1e-2
    x[:, 700] *= tail / 1e-2
    x[1] = rng.standard_normal(1024)      # a row of the same launch whose guess is right
    xd = torch.from_numpy(x).to(dt).cuda()
    y = torch.zeros((3, 100), device="cuda")
    W = b2q.WeightQ4(b, 100, 1024)
    b2q.mul_vec_q4(W, xd, 3, y)
    x64 = xd.double().cpu().numpy()
    within(y.double().cpu().numpy(), x64 @ w.T, (32 + 32 + 8) * 2.0 ** -23 * (np.abs(x64) @ mag.T)
           + 2.0 ** -29 * np.abs(x64).max(1, keepdims=True) * mag.sum(1)[None])


def test_zero_rows():
    rng = np.random.default_rng(12)
    b, _, _ = blocks(rng, 50, 320, Q4_1)
    W = b2q.WeightQ4(b, 50, 320, Q4_1)
    for dt in (F32, F16, BF16):
        y = torch.ones((2, 50), dtype=dt, device="cuda")
        b2q.mul_vec_q4(W, torch.zeros((2, 320), dtype=dt, device="cuda"), 2, y)
        assert (y == 0).all()


def test_infinite_and_nan_activations_reach_the_result():
    rng = np.random.default_rng(0)
    b, w, _ = blocks(rng, 40, 64, Q4_0)
    W = b2q.WeightQ4(b, 40, 64)
    x = torch.ones((3, 64), device="cuda")
    x[1, 5], x[2, 40] = float("inf"), float("nan")
    y = torch.zeros((3, 40), device="cuda")
    b2q.mul_vec_q4(W, x, 3, y)
    y = y.cpu().numpy()
    assert np.isfinite(y[0]).all() and np.isnan(y[2]).all()
    sign = np.sign(w[:, 5])
    assert (y[1][sign > 0] == np.inf).all() and (y[1][sign < 0] == -np.inf).all() and np.isnan(y[1][sign == 0]).all()


def test_zero_scale_blocks_give_zeros():
    b = np.zeros((33, 3, 18), np.uint8)
    b[..., 2:] = 0xF0
    y = torch.ones((1, 33), device="cuda")
    b2q.mul_vec_q4(b2q.WeightQ4(b, 33, 96), torch.ones((1, 96), device="cuda"), 1, y)
    assert (y == 0).all()


@pytest.mark.parametrize("typ", [Q4_0, Q4_1], ids=["q4_0", "q4_1"])
def test_formats_against_gguf(typ, tmp_path):
    """Weights quantized and written by gguf-py, read through b2q_gguf, equal its decoder's."""
    gguf = pytest.importorskip("gguf")
    qt = gguf.GGMLQuantizationType.Q4_0 if typ == Q4_0 else gguf.GGMLQuantizationType.Q4_1
    rng = np.random.default_rng(2)
    q = gguf.quants.quantize(rng.standard_normal((48, 128)).astype(np.float32), qt)
    out = gguf.GGUFWriter(str(tmp_path / "w.gguf"), "test")
    out.add_tensor("w.weight", q, raw_dtype=qt)
    out.write_header_to_file()
    out.write_kv_data_to_file()
    out.write_tensors_to_file()
    out.close()
    import ctypes as C
    g = b2q.Gguf(tmp_path / "w.gguf")
    (name, t, ne, data), = g.tensors()
    assert (name, t, ne) == ("w.weight", typ, (128, 48))
    raw = np.ctypeslib.as_array((C.c_uint8 * q.nbytes).from_address(data))
    W = b2q.WeightQ4(raw, 48, 128, typ)
    w = gguf.quants.dequantize(q, qt).astype(np.float64)
    y = torch.zeros((2, 48), device="cuda")
    x = rng.standard_normal((2, 128)).astype(np.float32)
    b2q.mul_vec_q4(W, torch.from_numpy(x).cuda(), 2, y)
    within(y.double().cpu().numpy(), x.astype(np.float64) @ w.T, 44 * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) * 3)
    g.close()


def test_other_stream():
    check(2, 300, 512, stream=torch.cuda.Stream())


def test_no_rows():
    W = b2q.WeightQ4(np.zeros((4, 1, 18), np.uint8), 4, 32)
    b2q.mul_vec_q4(W, torch.zeros((0, 32), device="cuda"), 0, torch.zeros((0, 4), device="cuda"))


def test_refusals():
    raw = np.zeros((4, 2, 18), np.uint8)
    W = b2q.WeightQ4(raw, 4, 64)
    x, y = torch.zeros((2, 64), device="cuda"), torch.zeros((2, 4), device="cuda")
    b2q.mul_vec_q4(W, x, 2, y)
    bad = [
        (lambda: b2q.WeightQ4(raw, 4, 48), b2q.ERR_SHAPE),
        (lambda: b2q.WeightQ4(raw, 5, 64), b2q.ERR_SHAPE),
        (lambda: b2q.WeightQ4(raw, 4, 64, row_bytes=35), b2q.ERR_SHAPE),
        (lambda: b2q.WeightQ4(raw, 4, 32, b2q.GGML_Q8_0), b2q.ERR_INVALID),
        (lambda: b2q.mul_vec_q4(W, x[:, :32], 2, y), b2q.ERR_SHAPE),
        (lambda: b2q.mul_vec_q4(W, x.double(), 2, y), b2q.ERR_INVALID),
        (lambda: b2q.mul_vec_q4(W, x.half(), 2, y.bfloat16()), b2q.ERR_INVALID),
        (lambda: b2q.mul_vec_q4(W, x, 3, y), b2q.ERR_SHAPE),
        (lambda: b2q.mul_vec_q4(W, x, 2, y[:, :3]), b2q.ERR_SHAPE),
        (lambda: b2q.mul_vec_q4(W, x, 2, y, bias=torch.zeros(3, device="cuda")), b2q.ERR_SHAPE),
        (lambda: b2q.mul_vec_q4(W, x, 2, y, residual=y.half()), b2q.ERR_SHAPE),
    ]
    for call, status in bad:
        with pytest.raises(b2q.B2QError) as e:
            call()
        assert e.value.status == status
    assert b2q.lib().b2q_mul_vec_q4(None, None, 0, 1, 32, 32, None, 0, 4, None, None, None) == b2q.ERR_INVALID
    assert b2q.lib().b2q_weight_q4_release(None) == b2q.OK


@pytest.mark.parametrize("m, k, typ, dt", [(4, 8640, Q4_1, F32), (3, 12800, Q4_0, F32), (8, 12800, Q4_0, F32),
                                           (7, 9600, Q4_1, BF16), (9, 14336, Q4_0, F16)])
def test_long_rows_that_fill_shared_memory(m, k, typ, dt):
    check(m, 70, k, typ, dt, bias=True)


@pytest.mark.parametrize("typ", [Q4_0, Q4_1], ids=["q4_0", "q4_1"])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("at", [3, 700])
def test_values_beside_a_far_larger_one(typ, dt, at):
    """A value that no weight takes part in, up to 1e7 times the others (3e4 in fp16): what they
    keep is 2^-34 of it, as the header says, and 2^-23 of themselves.  An X of 32 columns is held
    within 2^-29 of it, which is 2^-34 a column again."""
    rng = np.random.default_rng(21)
    b, w, mag = blocks(rng, 200, 1152, typ)
    blk, i = at // 32, at % 32
    head = 2 if typ == Q4_0 else 4
    nib = b[:, blk, head + i % 16]
    zero = 8 if typ == Q4_0 else 0
    b[:, blk, head + i % 16] = (nib & 0xF0) | zero if i < 16 else (nib & 0x0F) | zero << 4
    w[:, at] = mag[:, at] = 0.0
    if typ == Q4_1:      # ... nor the block's minimum
        cols = slice(blk * 32, blk * 32 + 32)
        m = b[:, blk, 2:4].copy().view(np.float16).astype(np.float64)
        w[:, cols] -= m
        w[:, at] = 0.0
        mag[:, cols] -= np.abs(m)
        mag[:, at] = 0.0
        b[:, blk, 2:4] = 0
    W = b2q.WeightQ4(b, 200, 1152, typ)
    sizes = (1e2, 1e3, 1e4, 3e4) if dt == F16 else (1e2, 1e4, 1e5, 1e6, 1e7)
    x = rng.standard_normal((len(sizes), 1152)).astype(np.float32)
    x[:, at] = sizes
    xd = torch.from_numpy(x).to(dt).cuda()
    y = torch.zeros((len(sizes), 200), device="cuda")
    b2q.mul_vec_q4(W, xd, len(sizes), y)
    x64 = xd.double().cpu().numpy()
    tol = (32 + 36 + 8 + 1) * 2.0 ** -23 * (np.abs(x64) @ mag.T) \
        + 2.0 ** -34 * np.abs(x64).max(1, keepdims=True) * mag.sum(1)[None]
    within(y.double().cpu().numpy(), x64 @ w.T, tol)
    W.release()


def test_a_row_of_one_scale_keeps_its_last_bits():
    # one weight of 1 in each row of them: the result is the activation as it is held
    k = 64
    b = np.zeros((k, k // 32, 18), np.uint8)
    b[..., 2:] = 0x88
    for n in range(k):
        b[n, n // 32, :2] = np.float16(1.0).view(np.uint16).reshape(1).view(np.uint8)
        i = n % 32
        b[n, n // 32, 2 + i % 16] = 0x89 if i < 16 else 0x98
    W = b2q.WeightQ4(b, k, k)
    rng = np.random.default_rng(22)
    x = (rng.standard_normal((16, k)) * 2.0 ** rng.uniform(-30, 0, (16, k))).astype(np.float32)
    x[:, 40] = 1.5
    for dt, own in ((F32, 2.0 ** -23), (F16, 0.0), (BF16, 0.0)):
        xd = torch.from_numpy(x).to(dt).cuda()
        y = torch.zeros((16, k), device="cuda")
        b2q.mul_vec_q4(W, xd, 16, y)
        x64 = xd.double().cpu().numpy()
        within(y.double().cpu().numpy(), x64, own * np.abs(x64) + 2.0 ** -34 * np.abs(x64).max(1, keepdims=True))
