"""b2q_attention_paged against softmax attention in 64 bits.

Tolerance, from the arithmetic.  A score is an fp32 sum of d products of 16-bit
values: off by at most delta = (d + 8) 2^-24 scale sum|q k|, and its exponential
by that and by the rounding of its argument, 2^-22 (|s| + |max|).  Probabilities
and their sum carry these relative errors, so a result is off by at most
(2 delta + 2^-22 (|s| + |max|) + c) sum p|v|, where c covers the sums over the
keys (chains of at most n / 16 + 64 additions of 2^-23) and what the products
with V may round of a probability (2^-20 where the result keeps 32 bits, 2^-15
where it is rounded to 16).  Then one rounding to the output's type.
"""
import numpy as np
import pytest

import b2q
from decode_util import TINY, UNIT, deal_pages, device, i32, within

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN = float("nan")


@pytest.fixture(scope="module", autouse=True)
def dev():
    device()


def reference(q, keys, vals, scale):
    """One row: q [hq][d], keys/vals [n][hk][d] -> out, lse, tolerance without the final rounding."""
    hq, d = q.shape
    n, hk = keys.shape[:2]
    out, lse, tol, ltol = np.zeros((hq, d)), np.full(hq, -np.inf), np.zeros((hq, d)), np.zeros(hq)
    if n == 0:
        return out, lse, tol, ltol
    for h in range(hq):
        k, v = keys[:, h // (hq // hk)], vals[:, h // (hq // hk)]
        s = k @ q[h] * scale
        m = s.max()
        p = np.exp(s - m)
        z = p.sum()
        out[h], lse[h] = (p / z) @ v, m + np.log(z)
        delta = (d + 8) * 2.0 ** -24 * scale * (np.abs(k) @ np.abs(q[h])) + 2.0 ** -22 * (np.abs(s) + abs(m))
        # keys far below the maximum move nothing: their errors count with their weight
        rel = 2 * max((p / z) @ delta, delta[p > 1e-3].max(initial=0.0)) + (n / 16 + 64) * 2.0 ** -23
        tol[h] = rel * ((p / z) @ np.abs(v))
        ltol[h] = rel + 2.0 ** -22 * (abs(lse[h]) + 1)
    return out, lse, tol, ltol


def check(lens, hq, hk, d, dt, out_dt=F32, page=16, window=0, seq_of=None, scale=None, nhd=False, spread=1.0,
          want_lse=True, scratch=None, stream=None, q_pad=0, mean=0.0, n_pages=None):
    rng = np.random.default_rng(sum(lens) + hq * 31 + d)
    rows = len(lens)
    if seq_of is None:
        owner, table_lens = list(range(rows)), lens
    else:
        owner = seq_of
        table_lens = [max([0] + [x for x, s in zip(lens, seq_of) if s == i]) for i in range(max(seq_of) + 1)]
    table, pages = deal_pages(rng, table_lens, page, n_pages=n_pages)
    shape = (pages, page, hk, d) if nhd else (pages, hk, page, d)
    # whatever no request owns is NaN: behind a length, in a last page, in free pages
    kc, vc = (torch.full(shape, NAN, dtype=dt, device="cuda") for _ in range(2))
    if nhd:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    keys, vals = [], []
    for i, n in enumerate(table_lens):
        k, v = (torch.from_numpy(rng.standard_normal((n, hk, d)).astype(np.float32)).to(dt) for _ in range(2))
        if n:
            j = np.arange(n)
            pg, row = torch.from_numpy(table[i, j // page].astype(np.int64)), torch.from_numpy(j % page)
            kc[pg.cuda(), :, row.cuda()] = k.cuda()
            vc[pg.cuda(), :, row.cuda()] = v.cuda()
        keys.append(k.double().numpy())
        vals.append(v.double().numpy())
    q = torch.from_numpy((mean + spread * rng.standard_normal((rows, hq * d + q_pad))).astype(np.float32)).to(dt)
    qd = q.cuda()[:, :hq * d]
    out = torch.full((rows, hq * d + 8), NAN, dtype=out_dt, device="cuda")
    lse = torch.full((rows, hq), NAN, dtype=F32, device="cuda") if want_lse else None
    cache = b2q.KVCache(kc, vc)
    scratch = b2q.attention_paged_scratch(hq, cache) if scratch is None else scratch
    torch.cuda.synchronize()
    b2q.attention_paged(qd, cache, torch.from_numpy(table).cuda(), i32(lens), out[:, :hq * d], scratch,
                        seq_of=None if seq_of is None else i32(seq_of), scale=scale, window=window, lse=lse,
                        stream=stream)
    torch.cuda.synchronize()
    assert b2q.check_device() == 0
    assert torch.isnan(out[:, hq * d:].float()).all()
    got = out[:, :hq * d].double().cpu().numpy().reshape(rows, hq, d)
    more = 2.0 ** -20 if out_dt == F32 else 2.0 ** -15
    for r in range(rows):
        n = lens[r] if owner[r] >= 0 else 0
        lo = max(0, n - window) if window else 0
        o = max(owner[r], 0)
        ref, rl, tol, lt = reference(q[r, :hq * d].double().numpy().reshape(hq, d), keys[o][lo:n], vals[o][lo:n],
                                     d ** -0.5 if scale is None else scale)
        av = np.abs(vals[o][lo:n]).max(axis=0).repeat(hq // hk, 0) if n > lo else 0.0
        within(got[r], ref, tol + more * av + UNIT[out_dt] * 1.01 * np.abs(ref) + TINY[out_dt])
        if want_lse:
            gl = lse[r].double().cpu().numpy()
            if n > lo:
                within(gl, rl, lt)
            else:
                assert (gl == -np.inf).all() and (got[r] == 0).all()
    return out


@pytest.mark.parametrize("dt, out_dt", [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 80, 96, 104, 128, 192, 256])
def test_types_and_head_widths(dt, out_dt, d):
    check([1, 70, 0, 333], 4, 2, d, dt, out_dt)


@pytest.mark.parametrize("hq, hk", [(1, 1), (16, 16), (3, 1), (8, 8), (10, 2), (28, 4), (8, 1), (16, 1), (17, 1), (40, 2),
                                    (64, 1)])
def test_head_groups(hq, hk):
    check([65, 1, 200], hq, hk, 64, F16, F32)
    check([129, 31], hq, hk, 128, BF16, BF16)


@pytest.mark.parametrize("page", [1, 2, 8, 16, 32, 128, 1024])
def test_lengths_around_tiles_and_pages(page):
    check([0, 1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1023, 1024, 1025], 4, 2, 64,
          F16, F32, page=page)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 1000, 100000])
def test_windows(window):
    check([0, 1, 14, 16, 99, 100, 101, 700, 1500], 6, 2, 80, F16, F32, window=window, page=8)


def test_one_long_request_is_split_and_joined():
    check([20011], 8, 1, 128, F16, F32, page=64)
    check([20011], 5, 5, 72, BF16, BF16, page=16)


def test_ragged_batch():
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 900, 150).tolist()
    lens[7] = 6000
    check(lens, 8, 2, 64, F16, F16, page=16)


def test_more_rows_than_a_wave_of_short_ones():
    check([(i * 7) % 20 for i in range(3000)], 2, 1, 64, F16, F32, page=16, want_lse=False)


def test_causal_rows_of_shared_requests():
    # a prompt's rows: each reads its request's keys up to itself; idle rows between
    seq_of = [0] * 20 + [-1, 1, 1, -1] + [2] * 3
    lens = list(range(1, 21)) + [5, 40, 41, 0] + [3, 100, 7]
    check(lens, 4, 2, 64, F16, F32, seq_of=seq_of)


def test_cache_orders_and_query_strides():
    check([100, 3, 40], 4, 2, 64, F16, F32, nhd=True)
    check([100, 3, 40], 4, 2, 72, BF16, BF16, nhd=True, page=8, q_pad=16)


def test_scores_that_span_the_type():
    check([300, 77], 8, 2, 128, F16, F32, spread=12.0)      # scores of hundreds: one key takes it all
    check([300, 77], 8, 2, 128, F16, F32, scale=0.0)        # all keys alike
    check([300, 77], 8, 2, 64, F16, F32, scale=-0.3)        # a negative scale turns the order round
    check([257], 8, 2, 64, BF16, F32, scale=2.0, mean=3.0)


def test_lowest_value_scores_stay_finite():
    # every score is hugely negative, later ones even more: no row may come out empty
    k = torch.full((2, 1, 16, 64), -200.0, dtype=F16, device="cuda")
    k[1] = -220.0
    v = torch.ones((2, 1, 16, 64), dtype=F16, device="cuda")
    v[1] = 5.0
    q = torch.full((1, 64), 200.0, dtype=F16, device="cuda")
    c = b2q.KVCache(k, v)
    out, lse = torch.empty((1, 64), device="cuda"), torch.empty((1, 1), device="cuda")
    b2q.attention_paged(q, c, i32([0, 1]).view(1, 2), i32([32]), out, b2q.attention_paged_scratch(1, c), scale=1.0,
                        lse=lse)
    torch.cuda.synchronize()
    assert (out == 1.0).all() and abs(lse.item() - (-200.0 * 200 * 64 + np.log(16))) < 1.0


def test_bits_repeat_and_scratch_is_left_clean():
    cache = b2q.KVCache(*(torch.zeros((1, 2, 16, 128), dtype=F16, device="cuda") for _ in range(2)))
    scratch = b2q.attention_paged_scratch(8, cache)
    a = check([5000, 17, 900], 8, 2, 128, F16, F32, scratch=scratch)
    check([9], 8, 2, 128, F16, F32, scratch=scratch)
    check([40] * 700, 8, 2, 128, F16, F32, scratch=scratch, want_lse=False)
    b = check([5000, 17, 900], 8, 2, 128, F16, F32, scratch=scratch)
    assert torch.equal(a[:, :1024], b[:, :1024])


def test_other_stream():
    s = torch.cuda.Stream()
    check([800, 40], 8, 2, 128, F16, F32, stream=s)


def test_offsets_past_32_bits():
    # pages behind element 2^32: K and V share one buffer of 9 GB
    d, hk, page = 128, 8, 64
    n_pages = (2 ** 32 + 2 ** 27) // (d * hk * page)
    buf = torch.empty((n_pages, hk, page, d), dtype=F16, device="cuda")
    rng = np.random.default_rng(1)
    ids = [n_pages - 1, 3, n_pages - 5]
    vals = torch.from_numpy(rng.standard_normal((3, hk, page, d)).astype(np.float32)).half()
    buf[ids] = vals.cuda()
    n = 2 * page + 11
    q = torch.from_numpy(rng.standard_normal((1, 2 * hk * d)).astype(np.float32)).half()
    out = torch.empty((1, 2 * hk * d), device="cuda")
    c = b2q.KVCache(buf, buf)
    b2q.attention_paged(q.cuda(), c, i32(ids).view(1, 3), i32([n]), out, b2q.attention_paged_scratch(2 * hk, c))
    assert b2q.check_device() == 0
    kv = vals.double().numpy().transpose(0, 2, 1, 3).reshape(3 * page, hk, d)[:n]
    ref, _, tol, _ = reference(q.double().numpy().reshape(2 * hk, d), kv, kv, d ** -0.5)
    within(out.double().cpu().numpy().reshape(2 * hk, d), ref, tol + 2.0 ** -20 * 5 + 2.0 ** -23 * np.abs(ref))


def test_out_of_range_is_reported_and_left_out():
    k, v = (torch.ones((4, 1, 16, 64), dtype=F16, device="cuda") for _ in range(2))
    v[3] = 3.0
    c = b2q.KVCache(k, v)
    q = torch.ones((3, 64), dtype=F16, device="cuda")
    scratch = b2q.attention_paged_scratch(1, c)
    table = i32([0, 3, 1, 2]).view(2, 2)

    def call(tab, lens, seq_of):
        out = torch.full((3, 64), NAN, device="cuda")
        b2q.attention_paged(q, c, tab, i32(lens), out, scratch, seq_of=i32(seq_of))
        torch.cuda.synchronize()
        return out

    for tab, lens, seq_of, want in [
            (i32([0, 4, 1, 2]).view(2, 2), [32, 16, 32], [0, 1, 1], [1.0, 1.0, 1.0]),    # page 4 of 4
            (i32([0, -1, 1, 2]).view(2, 2), [32, 16, 32], [0, 1, 1], [1.0, 1.0, 1.0]),
            (table, [32, 33, 32], [0, 1, 1], [2.0, 1.0, 1.0]),                           # past the table
            (table, [32, -1, 32], [0, 1, 1], [2.0, 0.0, 1.0]),
            (table, [32, 16, 32], [0, 2, 1], [2.0, 0.0, 1.0]),                           # no such request
            (table, [32, 16, 32], [0, -2, 1], [2.0, 0.0, 1.0])]:
        out = call(tab, lens, seq_of)
        with pytest.raises(b2q.B2QError) as e:
            b2q.check_device()
        assert "code 7" in str(e.value)
        assert torch.allclose(out, torch.tensor(want, device="cuda")[:, None].expand(3, 64), atol=1e-6)
    call(table, [32, 16, 0], [0, 1, -1])
    assert b2q.check_device() == 0


def test_no_rows():
    c = b2q.KVCache(*(torch.zeros((1, 1, 16, 64), dtype=F16, device="cuda") for _ in range(2)))
    b2q.attention_paged(torch.zeros((0, 64), dtype=F16, device="cuda"), c, i32([]).view(0, 1), i32([]),
                        torch.zeros((0, 64), device="cuda"), b2q.attention_paged_scratch(1, c))


def test_refusals():
    k, v = (torch.zeros((2, 2, 16, 64), dtype=F16, device="cuda") for _ in range(2))
    c = b2q.KVCache(k, v)
    q, out = torch.zeros((2, 256), dtype=F16, device="cuda"), torch.zeros((2, 256), device="cuda")
    table, lens, scratch = i32([0, 1]).view(2, 1), i32([1, 1]), b2q.attention_paged_scratch(4, c)
    b2q.attention_paged(q, c, table, lens, out, scratch)
    bad = [
        (lambda: b2q.attention_paged(q.bfloat16(), c, table, lens, out, scratch), b2q.ERR_SHAPE),
        (lambda: b2q.attention_paged(q, c, table, lens, out.bfloat16(), scratch), b2q.ERR_INVALID),
        (lambda: b2q.attention_paged(q, c, table, lens[:1], out, scratch), b2q.ERR_SHAPE),
        (lambda: b2q.attention_paged(q, c, table[:1], lens, out, scratch), b2q.ERR_SHAPE),
        (lambda: b2q.attention_paged(q, c, table.long(), lens, out, scratch), b2q.ERR_INVALID),
        (lambda: b2q.attention_paged(q, c, table, lens, out, scratch, window=-1), b2q.ERR_INVALID),
        (lambda: b2q.attention_paged(q, c, table, lens, out, scratch, scale=NAN), b2q.ERR_INVALID),
        (lambda: b2q.attention_paged(q[:, :192], c, table, lens, out[:, :192], scratch), b2q.ERR_SHAPE),
        (lambda: b2q.attention_paged(q, c, table, lens, out, scratch[:0]), b2q.ERR_SHAPE),
        (lambda: b2q.attention_paged_scratch(3, c), b2q.ERR_SHAPE),
    ]
    for call, status in bad:
        with pytest.raises(b2q.B2QError) as e:
            call()
        assert e.value.status == status
    null = b2q.lib().b2q_attention_paged(None, 256, 2, 4, c.ref, None, 1, 1, 2, None, None, 1.0, 0, None, 0, 256, None,
                                         None, None)
    assert null == b2q.ERR_INVALID
    assert b2q.check_device() == 0


@pytest.mark.parametrize("shape", [(5, 1, 16, 64), (5, 2, 1, 64), (1, 2, 16, 64), (1, 1, 1, 64)])
def test_dimensions_of_one_entry_may_have_any_stride(shape):
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(shape, generator=g).half().cuda() for _ in range(2))
    q, lens = torch.randn((1, shape[1] * 64), generator=g).half().cuda(), i32([shape[0] * shape[2]])
    table = i32(range(shape[0])).view(1, -1)
    outs = []
    for st in (None, 3, 0, 65):     # legal strides of such a dimension, none of a legal cache row
        kv = [t if st is None else t.as_strided(shape, [st if n == 1 else s for n, s in zip(shape, t.stride())])
              for t in (k, v)]
        c = b2q.KVCache(*kv)
        outs.append(torch.full((1, shape[1] * 64), NAN, device="cuda"))
        b2q.attention_paged(q, c, table, lens, outs[-1], b2q.attention_paged_scratch(shape[1], c))
    b2q.KVCache(k, kv[1])
    assert b2q.check_device() == 0
    assert torch.isfinite(outs[0]).all() and all(torch.equal(outs[0], o) for o in outs)


def test_scratch_that_is_not_contiguous_is_refused():
    # an expanded view has the entries, not the bytes
    c = b2q.KVCache(*(torch.zeros((2, 2, 16, 64), dtype=F16, device="cuda") for _ in range(2)))
    q, out = torch.zeros((1, 256), dtype=F16, device="cuda"), torch.zeros((1, 256), device="cuda")
    n = b2q.attention_paged_scratch(4, c).numel()
    buf = torch.zeros(2 * n, dtype=torch.uint8, device="cuda")
    b2q.attention_paged(q, c, i32([0]).view(1, 1), i32([1]), out, buf)
    for scratch in (buf[:1].expand(n), buf[::2], buf.view(2, n)[:, :n // 2 + 8]):
        with pytest.raises(b2q.B2QError) as e:
            b2q.attention_paged(q, c, i32([0]).view(1, 1), i32([1]), out, scratch)
        assert e.value.status == b2q.ERR_SHAPE


@pytest.mark.parametrize("lens", [[5000], [2000, 2100, 1900], [9001], [20011, 3, 700]])
@pytest.mark.parametrize("hq, hk, d", [(16, 16, 72), (8, 8, 64), (8, 4, 64), (3, 1, 96), (4, 2, 128), (6, 6, 192), (8, 8, 256)])
def test_bits_repeat_whoever_reports_last(hq, hk, d, lens):
    # a CTA may come to join one group or two: the order of a group's sums must not know
    g = torch.Generator(device="cuda").manual_seed(sum(lens) + d)
    table, pages = deal_pages(np.random.default_rng(4), lens, 16)
    c = b2q.KVCache(*(torch.randn(pages, hk, 16, d, device="cuda", generator=g).half() for _ in range(2)))
    q = torch.randn(len(lens), hq * d, device="cuda", generator=g).half()
    table, lens, scratch = torch.from_numpy(table).cuda(), i32(lens), b2q.attention_paged_scratch(hq, c)
    outs = [torch.empty(q.shape, device="cuda") for _ in range(100)]
    for out in outs:
        b2q.attention_paged(q, c, table, lens, out, scratch)
    torch.cuda.synchronize()
    assert sum(not torch.equal(outs[0], o) for o in outs) == 0 and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("dt, out_dt", [(F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("hq, hk, d, lens, window", [(4, 2, 64, [1, 33, 200, 0], 0), (16, 16, 72, [997, 40], 0),
                                                     (8, 1, 256, [700, 3000], 500), (20, 1, 128, [2500, 7], 0),
                                                     (3, 3, 96, [20, 6001], 0)])
def test_infinite_and_nan_values_reach_the_result(dt, out_dt, hq, hk, d, lens, window):
    # a value of +inf or -inf with weight is the result, both signs and NaN are NaN; other
    # columns, heads and rows keep their sums, and what lies outside the window is not read
    rng = np.random.default_rng(hq + d)
    table, pages = deal_pages(rng, lens, 16)
    kc, vc = (torch.full((pages, hk, 16, d), NAN, dtype=dt, device="cuda") for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((len(lens), hq * d)).astype(np.float32)).to(dt)
    keys, vals, inf = [], [], float("inf")
    for i, n in enumerate(lens):
        k, v = (torch.from_numpy(rng.standard_normal((n, hk, d)).astype(np.float32)).to(dt) for _ in range(2))
        lo = max(0, n - window) if window else 0
        if n:
            at = lambda: int(rng.integers(lo, n))
            v[at(), 0, 1] = inf
            v[at(), 0, 2] = -inf
            v[n - 1, hk - 1, 5] = inf
            v[lo, hk - 1, 5] = inf
            v[at(), hk - 1, 8] = NAN
            v[at(), hk - 1, 8] = inf if n > 1 else NAN
            if n > lo + 1:
                v[lo, 0, 11], v[n - 1, 0, 11] = inf, -inf
            v[at(), 0, d - 1] = -inf
            if lo:
                v[lo - 1, 0, 20] = inf
            j = np.arange(n)
            pg, row = torch.from_numpy(table[i, j // 16].astype(np.int64)).cuda(), torch.from_numpy(j % 16).cuda()
            kc[pg, :, row], vc[pg, :, row] = k.cuda(), v.cuda()
        keys.append(k.double().numpy())
        vals.append(v.double().numpy())
    out = torch.zeros((len(lens), hq * d), dtype=out_dt, device="cuda")
    c = b2q.KVCache(kc, vc)
    scratch = b2q.attention_paged_scratch(hq, c)
    lse = torch.zeros((len(lens), hq), device="cuda")
    for _ in range(2):          # (the second time on scratch that has seen them)
        b2q.attention_paged(q.cuda(), c, torch.from_numpy(table).cuda(), i32(lens), out, scratch, window=window, lse=lse)
    assert b2q.check_device() == 0
    got = out.double().cpu().numpy().reshape(len(lens), hq, d)
    more = 2.0 ** -20 if out_dt == F32 else 2.0 ** -15
    for r, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        k, v = keys[r][lo:n], vals[r][lo:n]
        plain = np.where(np.isfinite(v), v, 0.0)
        ref, rl, tol, lt = reference(q[r].double().numpy().reshape(hq, d), k, plain, d ** -0.5)
        per = hq // hk
        up, down, nan = (f(v).any(0).repeat(per, 0) if n else np.zeros((hq, d), bool)
                         for f in (np.isposinf, np.isneginf, np.isnan))
        nan |= up & down
        np.testing.assert_array_equal(np.isnan(got[r]), nan)
        np.testing.assert_array_equal(np.isposinf(got[r]), up & ~nan)
        np.testing.assert_array_equal(np.isneginf(got[r]), down & ~nan)
        good = ~(up | down | nan)
        tol = tol + more * np.abs(plain).max(axis=0, initial=0.0).repeat(per, 0) + UNIT[out_dt] * 1.01 * np.abs(ref) \
            + TINY[out_dt]
        within(got[r][good], ref[good], tol[good])
        if n:
            within(lse[r].double().cpu().numpy(), rl, lt)


def test_scores_that_are_no_numbers_make_the_row_none():
    # a NaN or infinite key: no weight of the row is a number, whatever the values are
    k, v = (torch.ones((2, 1, 16, 64), dtype=F16, device="cuda") for _ in range(2))
    v[0, 0, 3, 7] = float("inf")
    q, c = torch.ones((2, 64), dtype=F16, device="cuda"), None
    for bad in (NAN, float("inf")):
        k[0, 0, 5, 9] = bad
        c = b2q.KVCache(k, v)
        out = torch.zeros((2, 64), device="cuda")
        b2q.attention_paged(q, c, i32([0, 1]).view(2, 1), i32([16, 16]), out, b2q.attention_paged_scratch(1, c))
        assert torch.isnan(out[0]).all() and (out[1] == 1.0).all()
    assert b2q.check_device() == 0


@pytest.mark.parametrize("d, page", [(64, 16), (256, 16), (256, 8), (192, 16)])
def test_the_longest_context_an_int32_counts(d, page):
    # 2^31 - page keys on five pages in turn, read through a window at their end
    blocks = (2 ** 31 - 1) // page
    n, window = blocks * page, 229
    rng = np.random.default_rng(d + page)
    k, v = (torch.from_numpy(rng.standard_normal((5, 1, page, d)).astype(np.float32)).half() for _ in range(2))
    table = (torch.arange(blocks, dtype=torch.int32, device="cuda") % 5).view(1, blocks)
    q = torch.from_numpy(rng.standard_normal((1, d)).astype(np.float32)).half()
    out = torch.empty((1, d), device="cuda")
    c = b2q.KVCache(k.cuda(), v.cuda())
    b2q.attention_paged(q.cuda(), c, table, i32([n]), out, b2q.attention_paged_scratch(1, c), window=window)
    assert b2q.check_device() == 0
    j = np.arange(n - window, n, dtype=np.int64)
    keys, vals = (t.double().numpy()[j // page % 5, :, j % page] for t in (k, v))
    ref, _, tol, _ = reference(q.double().numpy(), keys, vals, d ** -0.5)
    within(out.double().cpu().numpy(), ref, tol + 2.0 ** -20 * np.abs(vals).max(0) + 2.0 ** -24 * 1.01 * np.abs(ref))
