"""b2q_qk_norm_rope against its formula in 64 bits.

Tolerance, from the arithmetic: the mean of d squares in fp32 is off by at most
d units (2^-24) relatively, its root by half of that, and the scaling and the
rotation add a handful of roundings, all relative to |x_a| + |x_b| of the pair;
the result is rounded once to the output's type.
"""
import numpy as np
import pytest

import b2q
from decode_util import TINY, UNIT, device, i32, within

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def dev():
    device()


def reference(x, hq, hk, d, qw, kw, eps, table, pos, inter):
    """(heads [T][hq + 2 hk][d], the sum of absolute terms of each) in 64 bits."""
    T = x.shape[0]
    x = x.double().cpu().numpy().reshape(T, hq + 2 * hk, d)
    mag = np.abs(x)
    rot = 0 if table is None else table.shape[1]
    for h in range(hq + hk):
        w = qw if h < hq else kw
        if w is not None:
            f = w.double().cpu().numpy() / np.sqrt((x[:, h] ** 2).mean(1, keepdims=True) + eps)
            x[:, h] = x[:, h] * f
            mag[:, h] = np.abs(x[:, h])
    if rot:
        half = rot // 2
        cs = table.double().cpu().numpy()[pos]
        c, s = cs[:, None, :half], cs[:, None, half:]
        ia, ib = np.arange(half), np.arange(half) + half
        if inter:
            ia, ib = 2 * np.arange(half), 2 * np.arange(half) + 1
        a, b = x[:, :hq + hk, ia].copy(), x[:, :hq + hk, ib].copy()
        both = np.abs(a) + np.abs(b)
        x[:, :hq + hk, ia], x[:, :hq + hk, ib] = a * c - b * s, b * c + a * s
        mag[:, :hq + hk, ia] = mag[:, :hq + hk, ib] = both
    return x, mag


def check(T, hq, hk, d, rot, dt, cdt, page=16, inter=False, norm=True, seed=0, ld_pad=0, nhd=False, scale=1.0,
          stream=None, offset=0):
    rng = np.random.default_rng(seed + T * 7 + d)
    heads = hq + 2 * hk
    base = torch.from_numpy((rng.standard_normal((T, heads * d + ld_pad)) * scale).astype(np.float32)).to(dt)
    flat = torch.zeros(base.numel() + offset, dtype=dt, device="cuda")
    flat[offset:] = base.reshape(-1).cuda()
    x = flat[offset:].view(T, heads * d + ld_pad)[:, :heads * d]
    qw, kw = (torch.from_numpy((1 + 0.3 * rng.standard_normal(d)).astype(np.float32)).cuda() if norm else None
              for _ in range(2))
    table = b2q.rope_table(5000, rot) if rot else None
    pos = rng.integers(0, 5000, T)
    pages = -(-T // page) + 2
    slot = rng.permutation(pages * page)[:T].copy()
    if T > 3:
        slot[2] = -1
    shape = (pages, page, hk, d) if nhd else (pages, hk, page, d)
    k, v = (torch.full(shape, 7.0, dtype=cdt, device="cuda") for _ in range(2))
    if nhd:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    q = torch.full((T, hq * d + 8), 9.0, dtype=cdt, device="cuda")[:, :hq * d]
    b2q.qk_norm_rope(x, hq, b2q.KVCache(k, v), q, i32(pos), i32(slot), qw, kw, 1e-5, table, inter, stream=stream)
    torch.cuda.synchronize()
    assert b2q.check_device() == 0
    ref, mag = reference(x, hq, hk, d, qw, kw, 1e-5, table, pos, inter)
    tol = UNIT[cdt] * np.abs(ref) * 1.01 + TINY[cdt] + (d / 2 + 8) * 2.0 ** -24 * mag
    within(q.double().cpu().numpy().reshape(T, hq, d), ref[:, :hq], tol[:, :hq])
    kept = slot >= 0
    pg, row = slot[kept] // page, slot[kept] % page
    for buf, at in ((k, hq), (v, hq + hk)):
        full = buf.double().cpu().numpy()
        within(full[pg, :, row], ref[kept][:, at:at + hk], tol[kept][:, at:at + hk])
        full[pg, :, row] = 7.0
        assert (full == 7.0).all(), "a slot that no row has was written"


@pytest.mark.parametrize("dt, cdt", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (F16, BF16)])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 80, 128, 200, 256])
def test_types_and_head_widths(dt, cdt, d):
    check(5, 6, 2, d, d, dt, cdt)
    check(3, 3, 3, d, d, dt, cdt, inter=True, norm=False)


@pytest.mark.parametrize("rot, d", [(0, 64), (2, 64), (6, 72), (32, 128), (36, 72), (64, 80), (126, 128)])
@pytest.mark.parametrize("inter", [False, True])
def test_partial_rotation(rot, d, inter):
    check(9, 4, 1, d, rot, F32, F16, inter=inter)
    check(9, 5, 5, d, rot, BF16, BF16, inter=inter, norm=False)


@pytest.mark.parametrize("T", [1, 2, 63, 1000])
@pytest.mark.parametrize("page", [1, 16, 1024])
def test_row_counts_and_pages(T, page):
    check(T, 8, 2, 128, 128, F16, F16, page=page)


def test_strides_orders_and_offsets():
    check(33, 4, 2, 64, 64, F32, F16, ld_pad=3)                  # rows not 16-byte aligned
    check(33, 4, 2, 64, 64, BF16, BF16, ld_pad=8, nhd=True)      # tokens before heads in a page
    check(33, 4, 2, 128, 128, F16, F16, offset=1)                # the first row is not aligned either
    check(33, 4, 2, 72, 72, F16, F16, offset=5, inter=True)


def test_large_and_small_values():
    check(17, 4, 2, 128, 128, F32, BF16, scale=1e15)             # squares stay finite in fp32
    check(17, 4, 2, 128, 128, F32, F16, scale=1e-3)
    check(17, 4, 2, 128, 128, F32, F16, scale=1e-3, norm=False)


def test_zero_head_stays_zero():
    k, v = (torch.ones((1, 1, 16, 64), dtype=F16, device="cuda") for _ in range(2))
    q = torch.ones((1, 64), dtype=F16, device="cuda")
    w = torch.ones(64, device="cuda")
    b2q.qk_norm_rope(torch.zeros((1, 192), device="cuda"), 1, b2q.KVCache(k, v), q, i32([3]), i32([5]), w, w, 0.0 + 1e-6,
                     b2q.rope_table(8, 64))
    torch.cuda.synchronize()
    assert (q == 0).all() and (k[0, 0, 5] == 0).all() and (v[0, 0, 5] == 0).all()


def test_queries_in_place():
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((50, 6 * 128)).astype(np.float32)).half().cuda()
    k, v, k2, v2 = (torch.zeros((4, 1, 16, 128), dtype=F16, device="cuda") for _ in range(4))
    pos, slot, table = i32(range(50)), i32(range(50)), b2q.rope_table(64, 128)
    w = torch.ones(128, device="cuda")
    q = torch.empty((50, 4 * 128), dtype=F16, device="cuda")
    b2q.qk_norm_rope(x, 4, b2q.KVCache(k, v), q, pos, slot, w, w, 1e-6, table)
    b2q.qk_norm_rope(x, 4, b2q.KVCache(k2, v2), x[:, :512], pos, slot, w, w, 1e-6, table)
    torch.cuda.synchronize()
    assert torch.equal(x[:, :512], q) and torch.equal(k, k2) and torch.equal(v, v2)


def test_padding_and_out_of_range_rows():
    rng = np.random.default_rng(4)
    x = torch.from_numpy(rng.standard_normal((4, 4 * 64)).astype(np.float32)).cuda()
    x[1] = float("nan")                                          # a padding row holds anything
    k, v = (torch.full((2, 1, 16, 64), 7.0, dtype=F16, device="cuda") for _ in range(2))
    q = torch.full((4, 128), 7.0, dtype=F16, device="cuda")
    b2q.qk_norm_rope(x, 2, b2q.KVCache(k, v), q, i32([0, -1, 2, 3]), i32([0, -1, -1, 31]), None, None, 1e-6,
                     b2q.rope_table(8, 64))
    assert b2q.check_device() == 0
    assert (q[1] == 0).all() and (k[1, 0, 15] != 7.0).any()
    for pos, slot in (([0, 8], [1, 2]), ([0, -2], [1, 2]), ([0, 1], [1, 32]), ([0, 1], [1, -2])):
        k.fill_(7.0)
        b2q.qk_norm_rope(x[2:], 2, b2q.KVCache(k, v), q[2:], i32(pos), i32(slot), None, None, 1e-6,
                         b2q.rope_table(8, 64))
        with pytest.raises(b2q.B2QError) as e:
            b2q.check_device()
        assert "code 6" in str(e.value)
        assert (k[0, 0, 1] != 7.0).any() and (k[0, 0, 2:] == 7.0).all() and (k[1] == 7.0).all()
    assert b2q.check_device() == 0


def test_other_stream():
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    check(40, 4, 2, 128, 128, F16, F16, stream=s)


def test_no_rows():
    k, v = (torch.zeros((1, 1, 16, 64), dtype=F16, device="cuda") for _ in range(2))
    b2q.qk_norm_rope(torch.zeros((0, 192), device="cuda"), 1, b2q.KVCache(k, v),
                     torch.zeros((0, 64), dtype=F16, device="cuda"), i32([]), i32([]))


def test_refusals():
    k, v = (torch.zeros((2, 2, 16, 64), dtype=F16, device="cuda") for _ in range(2))
    c = b2q.KVCache(k, v)
    x, q = torch.zeros((3, 8 * 64), device="cuda"), torch.zeros((3, 256), dtype=F16, device="cuda")
    pos, table = i32([0, 1, 2]), b2q.rope_table(8, 64)
    b2q.qk_norm_rope(x, 4, c, q, pos, pos, rope=table)
    bad = [
        (lambda: b2q.qk_norm_rope(x, 5, c, q, pos, pos, rope=table), b2q.ERR_SHAPE),
        (lambda: b2q.qk_norm_rope(x, 4, c, q.float(), pos, pos, rope=table), b2q.ERR_SHAPE),
        (lambda: b2q.qk_norm_rope(x.double(), 4, c, q, pos, pos, rope=table), b2q.ERR_INVALID),
        (lambda: b2q.qk_norm_rope(x, 4, c, q, pos[:2], pos, rope=table), b2q.ERR_SHAPE),
        (lambda: b2q.qk_norm_rope(x, 4, c, q, pos.long(), pos, rope=table), b2q.ERR_INVALID),
        (lambda: b2q.qk_norm_rope(x, 4, c, q, pos, pos, rope=b2q.rope_table(8, 128)), b2q.ERR_SHAPE),
        (lambda: b2q.qk_norm_rope(x, 4, c, q, pos, pos, torch.ones(63, device="cuda"), rope=table), b2q.ERR_SHAPE),
        (lambda: b2q.qk_norm_rope(x, 4, c, q, pos, pos, eps=-1.0, rope=table), b2q.ERR_INVALID),
        (lambda: b2q.qk_norm_rope(x, 4, b2q.KVCache(k.float(), v.float()), q.float(), pos, pos), b2q.ERR_INVALID),
        (lambda: b2q.KVCache(k, v[:1]), b2q.ERR_SHAPE),
    ]
    for call, status in bad:
        with pytest.raises(b2q.B2QError) as e:
            call()
        assert e.value.status == status
    for shape in [(2, 2, 12, 64), (2, 2, 2048, 64), (2, 2, 16, 60), (2, 2, 16, 264)]:
        z = torch.zeros(shape, dtype=F16, device="cuda")
        with pytest.raises(b2q.B2QError) as e:
            b2q.qk_norm_rope(torch.zeros((3, 8 * shape[3]), device="cuda"), 4, b2q.KVCache(z, z),
                             torch.zeros((3, 4 * shape[3]), dtype=F16, device="cuda"), pos, pos)
        assert e.value.status == b2q.ERR_SHAPE
    odd = torch.zeros(2 * 2 * 16 * 64 + 1, dtype=F16, device="cuda")[1:].view(2, 2, 16, 64)
    with pytest.raises(b2q.B2QError) as e:
        b2q.qk_norm_rope(x, 4, b2q.KVCache(odd, odd), q, pos, pos)
    assert e.value.status == b2q.ERR_ALIGN
    assert b2q.check_device() == 0
