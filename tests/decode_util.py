"""Inputs and 64-bit definitions shared by the tests of the decode operators."""
import numpy as np
import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
#: spacing of the subnormals, half of which a rounding may cost below the normal range
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def device():
    import pytest

    import b2q
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    b2q.init(0)


def cuda(a, dtype=None):
    t = a if isinstance(a, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(a))
    return t.to(dtype).cuda() if dtype is not None else t.cuda()


def i32(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def deal_pages(rng, lens, page, width=None, spare=3, n_pages=None):
    """Random distinct pages for each request: (table [n][width] int32 with
    unused entries far out of range, pages in all)."""
    need = [-(-int(x) // page) for x in lens]
    n_pages = n_pages or sum(need) + spare
    ids = rng.permutation(n_pages)[:sum(need)]
    width = width or max(need + [1])
    table = np.full((len(lens), width), 0x7FFFFFF0, np.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = ids[at:at + k]
        at += k
    return table, n_pages


def within(got, ref, tol):
    """Every |got - ref| <= tol (64-bit arrays); ref has no NaN."""
    got, ref, tol = (np.asarray(x, np.float64) for x in (got, ref, tol))
    assert got.shape == ref.shape
    assert np.isfinite(got).all(), "NaN or infinity in the result"
    over = np.abs(got - ref) - tol
    assert over.max(initial=-1.0) <= 0, (np.abs(got - ref).max(), over.max())
