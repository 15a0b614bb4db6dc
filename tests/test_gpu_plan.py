"""b2q_kv_plan against a request-by-request restatement: whole numbers, equal."""
import numpy as np
import pytest

import b2q
from decode_util import device, i32

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def dev():
    device()


def reference(ctx, new, page, free, table, rows):
    table = table.copy()
    width = table.shape[1]
    out = {k: np.full(rows, -1, np.int32) for k in ("seq", "pos", "slot")}
    out["len"] = np.zeros(rows, np.int32)
    t = taken = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        c, n = min(max(c, 0), width * page), max(n, 0)
        have, need = -(-c // page), min(-(-(c + n) // page), width)
        fresh = {}
        for b in range(have, need):
            fresh[b] = table[s, b] = free[taken] if taken < len(free) else -1
            taken += 1
        for i in range(n):
            if t < rows:
                p, b = c + i, (c + i) // page
                pg = fresh.get(b, table[s, b] if b < have else -1) if b < width else -1
                out["seq"][t], out["pos"][t], out["len"][t] = s, p, p + 1
                out["slot"][t] = pg * page + p % page if pg >= 0 else -1
            t += 1
    return table, out, [t, min(taken, len(free))]


def run(ctx, new, page, free, table, rows, stride=None):
    n, width = table.shape
    wide = np.full((n, stride or width), 77, np.int32)
    wide[:, :width] = table
    full = torch.from_numpy(wide).cuda()
    view = full[:, :width]
    out = {k: torch.full((rows,), 99, dtype=torch.int32, device="cuda") for k in ("seq", "pos", "slot", "len")}
    counts = torch.full((2,), 99, dtype=torch.int32, device="cuda")
    b2q.kv_plan(i32(ctx), i32(new), page, i32(free), view, out["seq"], out["pos"], out["slot"], out["len"], counts)
    torch.cuda.synchronize()
    assert (full[:, width:] == 77).all()
    return view.cpu().numpy(), {k: v.cpu().numpy() for k, v in out.items()}, counts.tolist()


def compare(ctx, new, page, width=None, spare=4, pad=0, n_free=None, rows=None, stride=None):
    rng = np.random.default_rng(len(ctx) * 1000 + page)
    need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    width = width or max(need + [1])
    ids = rng.permutation(sum(need) + spare + sum(-(-c // page) for c in ctx)).astype(np.int32)
    table = np.full((len(ctx), width), -1, np.int32)
    at = 0
    for i, c in enumerate(ctx):
        k = min(-(-c // page), width)
        table[i, :k] = ids[at:at + k]
        at += k
    free = ids[at:] if n_free is None else ids[at:at + n_free]
    rows = sum(new) + pad if rows is None else rows
    want = reference(ctx, new, page, free, table, rows)
    got = run(ctx, new, page, free, table, rows, stride)
    np.testing.assert_array_equal(got[0], want[0])
    for k in want[1]:
        np.testing.assert_array_equal(got[1][k], want[1][k], err_msg=k)
    assert got[2] == want[2]


@pytest.mark.parametrize("page", [1, 8, 16, 1024])
@pytest.mark.parametrize("ctx, new", [([0], [1]), ([5], [0]), ([15, 16, 17, 0], [1, 1, 1, 1]), ([0, 31, 100], [33, 0, 7]),
                                      ([0, 0, 0], [0, 0, 0]), ([3] * 40, [0] * 39 + [5])])
def test_small_steps(ctx, new, page):
    compare(ctx, new, page, pad=3)
    assert b2q.check_device() == 0


@pytest.mark.parametrize("n, hi", [(33, 1), (511, 40), (513, 3), (2000, 9), (16384, 1)])
def test_many_requests(n, hi):
    rng = np.random.default_rng(n)
    ctx = rng.integers(0, 200, n).tolist()
    new = rng.integers(0, hi + 1, n).tolist()
    compare(ctx, new, 16, stride=-(-240 // 16) + 9)
    assert b2q.check_device() == 0


def test_one_long_prompt_among_idle_requests():
    compare([7, 0, 40, 3], [0, 40001, 0, 1], 32)
    assert b2q.check_device() == 0


def test_no_requests_and_no_rows():
    _, out, counts = run([], [], 16, [], np.zeros((0, 4), np.int32), 5)
    assert counts == [0, 0] and (out["slot"] == -1).all() and (out["len"] == 0).all()
    compare([16, 3], [0, 0], 16, rows=0)
    assert b2q.check_device() == 0


@pytest.mark.parametrize("kw", [dict(n_free=2), dict(n_free=0), dict(width=2), dict(rows=20)],
                         ids=["pages", "no-pages", "table", "rows"])
def test_what_does_not_fit_is_reported(kw):
    compare([10, 0, 30], [20, 9, 3], 8, **kw)
    with pytest.raises(b2q.B2QError) as e:
        b2q.check_device()
    assert e.value.status == b2q.ERR_DEVICE and "code 8" in str(e.value)
    assert b2q.check_device() == 0


def test_hostile_lengths_are_reported():
    big = 2 ** 31 - 1
    ctx, new = [-5, big, 4, big], [3, big, -2, 1]
    table = np.zeros((4, 3), np.int32)
    got = run(ctx, new, 8, list(range(100, 140)), table, 50)
    want = reference([0, 24, 4, 24], [3, 47, 0, 0], 8, list(range(100, 140)), table, 50)
    for k in want[1]:
        np.testing.assert_array_equal(got[1][k], want[1][k], err_msg=k)
    with pytest.raises(b2q.B2QError):
        b2q.check_device()


def test_refusals():
    ok = dict(ctx=i32([1]), new=i32([1]), page=16, free=i32([0]), table=i32([0, 0]).view(1, 2),
              seq=i32([0]), pos=i32([0]), slot=i32([0]), len=i32([0]), counts=i32([0, 0]))

    def call(**kw):
        a = {**ok, **kw}
        b2q.kv_plan(a["ctx"], a["new"], a["page"], a["free"], a["table"], a["seq"], a["pos"], a["slot"], a["len"],
                    a["counts"])

    call()
    for kw, status in [(dict(page=0), b2q.ERR_SHAPE), (dict(page=24), b2q.ERR_SHAPE), (dict(page=2048), b2q.ERR_SHAPE),
                       (dict(new=i32([1, 2])), b2q.ERR_SHAPE), (dict(counts=i32([0])), b2q.ERR_SHAPE),
                       (dict(ctx=i32([1]).long()), b2q.ERR_INVALID), (dict(table=i32([0, 0])), b2q.ERR_SHAPE),
                       (dict(ctx=i32([1] * 16385), new=i32([1] * 16385), table=i32([0] * 16385).view(-1, 1)),
                        b2q.ERR_SHAPE)]:
        with pytest.raises(b2q.B2QError) as e:
            call(**kw)
        assert e.value.status == status, kw
    null = b2q.lib().b2q_kv_plan(None, None, 1, 16, None, 0, None, 1, 1, 1, None, None, None, None, None, None)
    assert null == b2q.ERR_INVALID
    assert b2q.check_device() == 0


@pytest.mark.parametrize("page", [1, 16, 1024])
def test_pages_whose_slots_would_wrap_are_no_pages(page):
    # slots are int32: 2^28 pages of 16 on, a page's slots would be those of page 0 again
    top = (2 ** 31 - 1) // page                 # the last page whose slots all fit
    table = np.full((3, 3), -1, np.int32)
    ctx, new = [page, page, 0], [page, 1, 1]
    table[:2, 0] = [7, 3]
    _, out, counts = run(ctx, new, page, [top - 1, top - 1, 5], table, page + 2)
    last = page + 1
    np.testing.assert_array_equal(out["slot"][:page], (top - 1) * page + np.arange(page))
    assert out["slot"][last] == 5 * page and counts == [page + 2, 3] and b2q.check_device() == 0
    if page == 1:
        return                                  # every int32 is a page of one token
    for bad in (top + 1, 2 ** 28, 2 ** 31 - 1):
        if bad <= top:
            continue
        got, out, counts = run(ctx, new, page, [bad, 9, 5], table, page + 2)
        assert (out["slot"][:page] == -1).all() and out["slot"][page] == 9 * page and out["slot"][last] == 5 * page
        np.testing.assert_array_equal(got, [[7, -1, -1], [3, 9, -1], [5, -1, -1]])
        with pytest.raises(b2q.B2QError) as e:
            b2q.check_device()
        assert "code 8" in str(e.value)
        # and one that the table holds already
        held = np.array([[bad, -1, -1]], np.int32)
        _, out, _ = run([1], [1], page, [4], held, 1)
        assert (out["slot"] == -1).all() and (out["pos"] == 1).all()
        with pytest.raises(b2q.B2QError):
            b2q.check_device()
