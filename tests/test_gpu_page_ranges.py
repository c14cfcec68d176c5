"""anygpu_copy_pages: caches without bytes lie anywhere, also inside of others."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("empty", ["no bytes", "no pages"])
@pytest.mark.parametrize("first", [False, True])
def test_empty_caches_inside_of_others(ops, empty, first):
    from anygpu_amd import capi
    pages = torch.arange(24, dtype=torch.int32, device="cuda").reshape(6, 4)
    to, origin = torch.tensor([0], dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda")
    at = pages.data_ptr()
    caches = [(at, 16, 6), (at + 16, 0 if empty == "no bytes" else 16, 6 if empty == "no bytes" else 0)]
    if first:
        caches.reverse()
    where = (ctypes.c_void_p * 2)(*[c[0] for c in caches])
    size, count = ((ctypes.c_int64 * 2)(*[c[k] for c in caches]) for k in (1, 2))
    rc = capi.load().anygpu_copy_pages(where, where, size, count, count, 2, to.data_ptr(), origin.data_ptr(), 1, torch.cuda.current_stream().cuda_stream)
    assert rc == capi.ANYGPU_OK
    assert torch.equal(pages[0], pages[5]) and pages[1, 0] == 4


def test_an_empty_source_inside_of_a_written_cache(ops):
    from anygpu_amd import capi
    pages = torch.arange(24, dtype=torch.int32, device="cuda").reshape(6, 4)
    to, origin = torch.tensor([1, 2], dtype=torch.int32, device="cuda"), torch.tensor([-1, 0], dtype=torch.int32, device="cuda")
    one = lambda kind, value: (kind * 1)(value)  # noqa: E731
    # (a source without pages: what is cleared is cleared, moves have nothing to take)
    rc = capi.load().anygpu_copy_pages(one(ctypes.c_void_p, pages.data_ptr()), one(ctypes.c_void_p, pages.data_ptr() + 16), one(ctypes.c_int64, 16), one(ctypes.c_int64, 6),
                                       one(ctypes.c_int64, 0), 1, to.data_ptr(), origin.data_ptr(), 2, torch.cuda.current_stream().cuda_stream)
    assert rc == capi.ANYGPU_OK
    assert not pages[1].any() and pages[2, 0] == 8


@pytest.mark.parametrize("moves,pages", [(5000, 12000), (20000, 60000), (3000, 90000), (4097, 4200)])
@pytest.mark.parametrize("apart", [True, False])
def test_lists_of_thousands_of_moves(ops, moves, pages, apart):
    gen = torch.Generator().manual_seed(moves)
    cache = torch.randn(pages, 12, generator=gen)
    if apart:
        order = torch.randperm(pages, generator=gen)
        to = order[:min(moves, pages // 2)]
        origin = order[len(to):][torch.randint(0, pages - len(to), (len(to),), generator=gen)]
        origin[::7] = -1
    else:
        to, origin = (torch.randint(-1, pages + 1, (moves,), generator=gen) for _ in range(2))
    want = cache.clone()
    for t, f in zip(to.tolist(), origin.tolist()):
        if 0 <= t < pages and -1 <= f < pages:
            want[t] = want[f].clone() if f >= 0 else 0.0
    got = cache.cuda()
    ops.tensor_copy_pages(got, got, to.int().cuda(), origin.int().cuda())
    assert torch.equal(got.cpu(), want)
