"""The selective scan of long sequences: blocks that walk many chunks, whole or in segments whose first pass is cut once more or not."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from scan_reference import check_scan, relative, selective_scan  # noqa: E402
from test_gpu_selective_scan import make, scan  # noqa: E402


# blocks: batch * heads * tiles of 64 rows; as many as the device has compute units (256) are not cut, 80 leave segments whose first pass goes over them whole, fewer
# leave segments that it takes in halves.  Rows end anywhere, and one is full.
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("batch,heads,dim,groups,size,seq,cut", [
    (4, 64, 64, 1, 64, 900, False), (2, 128, 64, 2, 16, 1001, False), (4, 64, 128, 1, 128, 700, False), (8, 32, 32, 1, 64, 833, False), (1, 256, 64, 4, 64, 1153, False),
    (2, 128, 40, 1, 130, 577, False),
    (1, 80, 64, 1, 64, 2500, True), (2, 40, 64, 2, 128, 2049, True), (1, 80, 32, 1, 64, 2111, True), (1, 80, 64, 1, 250, 1700, True),
    (1, 20, 64, 1, 64, 3001, True), (1, 8, 64, 1, 128, 4500, True),
])
def test_long_walks(ops, dtype, batch, heads, dim, groups, size, seq, cut):
    from anygpu_amd import capi
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert (capi.load().anygpu_selective_scan_workspace_bytes(batch, heads, dim, size, seq) > 0) == cut
    lengths = [seq, seq - 70, seq // 2, 0, 1, 64, seq // 3, seq - 1][:batch] if batch > 1 else None
    args = make(dtype, batch, heads, dim, groups, size, seq, seed=seq, lengths=lengths, std=0.7)
    y, state = scan(ops, args)
    check_scan(y, state, args)
    want, want_state = selective_scan(**args)
    # in the 2-norm: a rounding of the results and one of the weights or the state in front in half precision; float32: as in the short ones
    assert relative(y, want) <= (2.0 ** -11 if dtype == "f16" else 2.0 ** -20)
    assert relative(state, want_state) <= 2.0 ** -20
    for i in range(batch):
        n = seq if lengths is None else lengths[i]
        assert not y[i, n:].any()
        # the end of a row, where all that went wrong on the way has come together
        if n > 64:
            assert relative(y[i, n - 64:n], want[i, n - 64:n]) <= (2.0 ** -10.5 if dtype == "f16" else 2.0 ** -20), i


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("dim,size", [(33, 40), (16, 16), (64, 128)])
@pytest.mark.parametrize("chunks", range(1, 11))
def test_walks_of_every_length(ops, dtype, dim, size, chunks):
    # loops that go over two chunks at a time, with loads three ahead: they end after any number of them, in a whole chunk or anywhere in it
    for rest in (0, 1, 63):
        seq = 64 * chunks - rest
        args = make(dtype, 1, 256, dim, 2, size, seq, seed=seq, std=0.7)
        y, state = scan(ops, args)
        want, want_state = selective_scan(**args)
        assert relative(y, want) <= (2.0 ** -11 if dtype == "f16" else 2.0 ** -20), rest
        assert relative(state, want_state) <= 2.0 ** -20, rest
        assert relative(y[:, -1], want[:, -1]) <= (2.0 ** -10.5 if dtype == "f16" else 2.0 ** -20), rest
