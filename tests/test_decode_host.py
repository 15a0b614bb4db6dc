"""What the decode operators' binding and the decoder refuse or work out on the host: no GPU."""
import random

import pytest

import b2q
from b2q.decode import Decoder, entered_pages, placed_tokens

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("rows", [-1, 0, 9, 1000])
def test_a_step_refuses_rows_that_its_buffers_do_not_hold(rows):
    dec = Decoder.__new__(Decoder)   # before anything is looked up or launched
    dec.max_rows = 8
    with pytest.raises(b2q.B2QError) as e:
        dec.step(rows)
    assert e.value.status == b2q.ERR_SHAPE


def plan(ctx, new, page, n_free, width, rows):
    """seq_of, pos, slot of a step's rows as b2q_kv_plan gives them, token by token."""
    seq, pos, slot, taken = [-1] * rows, [-1] * rows, [-1] * rows, 0
    t = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        have = min(-(-c // page), width)
        for i in range(max(n, 0)):
            p = c + i
            if t < rows:
                seq[t], pos[t] = s, p
                first = taken + p // page - have
                if p // page < width and (p // page < have or first < n_free):
                    slot[t] = (1000 + first if p // page >= have else 50 * s + p // page) * page + p % page
            t += 1
        taken += max(min(-(-(c + max(n, 0)) // page), width) - have, 0)
    return seq, pos, slot


def test_tokens_without_a_row_or_a_page_do_not_count():
    rng = random.Random(3)
    for _ in range(300):
        n, page, rows = rng.randint(1, 6), rng.choice([1, 4, 16]), rng.randint(1, 40)
        ctx = [rng.randint(0, 40) for _ in range(n)]
        new = [rng.choice([0, 1, rng.randint(0, 30), -3]) for _ in range(n)]
        width, n_free = rng.randint(12, 60), rng.randint(0, 20)
        ctx = [min(c, width * page) for c in ctx]
        seq, pos, slot = plan(ctx, new, page, n_free, width, rows)
        count, last = placed_tokens(*(torch.tensor(v, dtype=torch.int32) for v in (seq, slot, new)))
        pages = {v // page for v in slot if v >= 1000 * page}       # taken in this step, and holding a token
        assert entered_pages(torch.tensor(slot, dtype=torch.int32), page) == len(pages)
        for s in range(n):
            good = [t for t in range(rows) if seq[t] == s and slot[t] >= 0]
            assert count[s] == len(good)
            assert 0 <= last[s] < rows          # an index that is always there to be read
            assert [pos[t] for t in good] == list(range(ctx[s], ctx[s] + len(good)))
            if good:
                assert last[s] == good[-1]


def test_a_released_request_leaves_no_hole_in_the_free_list():
    dec = Decoder.__new__(Decoder)
    dec.page_size = 16
    dec.table = torch.tensor([[4, 5, -1, 7], [1, -1, -1, -1], [6, 2, 3, -1]], dtype=torch.int32)
    dec.ctx_len = torch.tensor([64 + 20, 9, 48], dtype=torch.int32)     # the first one's past its table row
    dec.free = torch.tensor([0] + [-1] * 7, dtype=torch.int32)
    for s, free in [(0, [0, 4, 5, 7]), (2, [0, 4, 5, 7, 6, 2, 3]), (1, [0, 4, 5, 7, 6, 2, 3, 1]), (1, None)]:
        dec.release(s)
        assert dec.ctx_len[s] == 0 and (dec.table[s] == -1).all()
        if free:
            assert dec.free.tolist() == free + [-1] * (8 - len(free))
    assert sorted(dec.free.tolist()) == list(range(8))


@pytest.mark.parametrize("dim", [0, 1, 2])
def test_an_expanded_cache_is_refused(dim):
    # a stride of 0 reads as "contiguous order": the kernels would run past the tensor
    shape = [6, 4, 16, 64]
    shape[dim] = 1
    one = torch.zeros(shape, dtype=torch.float16)
    full = torch.zeros((6, 4, 16, 64), dtype=torch.float16)
    for k, v in ((one.expand(6, 4, 16, 64),) * 2, (one.expand(6, 4, 16, 64), full), (full, one.expand(6, 4, 16, 64))):
        with pytest.raises(b2q.B2QError) as e:
            b2q.KVCache(k, v)
        assert e.value.status == b2q.ERR_SHAPE
    b2q.KVCache(full, full)


def test_keys_and_values_on_two_devices_are_refused():
    k = torch.zeros((2, 4, 16, 64), dtype=torch.float16)
    v = torch.zeros((2, 4, 16, 64), dtype=torch.float16, device="meta")
    for pair in ((k, v), (v, k)):
        with pytest.raises(b2q.B2QError) as e:
            b2q.KVCache(*pair)
        assert e.value.status == b2q.ERR_INVALID


def test_weight_blocks_of_another_gpu_are_refused(monkeypatch):
    class Blocks:                               # a tensor of the second GPU, as far as it is looked at
        is_cuda, device = True, "cuda:1"
        numel, element_size, is_contiguous = (lambda self: 4 * 36), (lambda self: 1), (lambda self: True)
        get_device, data_ptr = (lambda self: 1), (lambda self: 4096)

    registered = []
    monkeypatch.setattr(b2q, "_device", lambda: 0)
    monkeypatch.setattr(b2q, "_stream", lambda s: None)
    monkeypatch.setattr(b2q.lib(), "b2q_weight_q4_register", lambda *a: registered.append(a) or 0)
    with pytest.raises(b2q.B2QError) as e:
        b2q.WeightQ4(Blocks(), 4, 64)
    assert e.value.status == b2q.ERR_INVALID and not registered
    monkeypatch.setattr(Blocks, "get_device", lambda self: 0)
    b2q.WeightQ4(Blocks(), 4, 64)
    assert len(registered) == 1


def test_a_native_half_that_does_not_load_is_left_out(monkeypatch, tmp_path):
    stale = tmp_path / "b2q_host.so"
    stale.write_bytes(b"\x7fELF of another time")
    monkeypatch.setattr(b2q, "HOST_PATH", stale)
    natives = ("_native_plan", "_native_rope", "_native_paged", "_native_vec")
    for n in natives:
        monkeypatch.setattr(b2q, n, b2q._not_native)
    for n in ("_plan", "_rope", "_paged", "_vec", "_device", "_raw_stream", "_INT32", "_F32"):
        monkeypatch.setattr(b2q, n, None)
    with pytest.warns(RuntimeWarning, match="does not load"):
        b2q._setup()
    assert b2q._plan is not None and b2q._vec is not None
    assert all(getattr(b2q, n) is b2q._not_native for n in natives)


def test_the_native_half_is_built_again_for_another_torch(tmp_path):
    import os
    import shutil
    import subprocess
    from pathlib import Path
    csrc = Path(b2q.__file__).resolve().parents[1] / "csrc"
    if not shutil.which("make"):
        pytest.skip("no make")
    stamp = tmp_path / "b2q_host.for"            # what b2q_host.so depends on

    def make(*more):
        subprocess.run(["make", "-s", "-C", str(csrc), f"OBJDIR={tmp_path}", str(stamp), *more], check=True)
        return stamp.read_text(), stamp.stat().st_mtime_ns

    first = make()
    assert torch.__version__ in first[0]
    os.utime(stamp, ns=(1, 1))
    assert make() == (first[0], 1)               # the same: not touched
    again = make("HOSTFOR=3.12.3 another torch")
    assert "another torch" in again[0] and again[1] > 1
    rules = (csrc / "Makefile").read_text()
    assert "../lib/b2q_host.so: b2q_host.cpp ../../include/b2q.h $(OBJDIR)/b2q_host.for" in rules
