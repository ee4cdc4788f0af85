"""Buffers that the feed-forward kernels write and read again at once: launch
after launch without a wait between them, two inputs in turn through the same
codes, scales, partial sums and packed rows.  Under programmatic dependent
launch several of these kernels are resident together."""

import math

import pytest
import torch

from test_gpu_feed_forward import BF16, F16, rand

pytestmark = pytest.mark.gpu

TURNS = 24


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("m,k", [(1, 32), (16, 1024), (33, 1001), (512, 4096), (4096, 7168)])
@pytest.mark.parametrize("dtype,code", [(BF16, 2), (F16, 1), (torch.float32, 0)])
def test_codes_written_and_read_in_turn(m, k, dtype, code):
    import dsv4_b200 as D
    from dsv4_b200 import _native as N
    xs = [rand(m, k, dtype=dtype, seed=s) * (1 + 2 * s) for s in (1, 2)]
    want = [D.restore_int8(D.checkpoint_int8(x)) for x in xs]
    k32 = -(-k // 32) * 32
    codes = torch.empty(m, k32, dtype=torch.int8, device="cuda")
    scales = torch.empty(k32 // 32, m, device="cuda")
    outs = torch.full((TURNS, m, k), 7.0, dtype=dtype, device="cuda")
    st = stream()
    torch.cuda.synchronize()
    for i in range(TURNS):
        N.call("dsv4_b200_checkpoint_int8", xs[i & 1].data_ptr(), code, m, k, k, codes.data_ptr(), scales.data_ptr(), st)
        N.call("dsv4_b200_restore_int8", codes.data_ptr(), scales.data_ptr(), m, k, outs[i].data_ptr(), code, k, st)
    for i in range(TURNS):
        assert torch.equal(outs[i], want[i & 1]), i
    # and on from what was restored: both kernels read what the one before them wrote
    a, b = xs[0].clone(), torch.empty_like(xs[0])
    for i in range(TURNS):
        N.call("dsv4_b200_checkpoint_int8", a.data_ptr(), code, m, k, k, codes.data_ptr(), scales.data_ptr(), st)
        N.call("dsv4_b200_restore_int8", codes.data_ptr(), scales.data_ptr(), m, k, b.data_ptr(), code, k, st)
        a, b = b, a
    step = xs[0]
    for i in range(TURNS):
        step = D.restore_int8(D.checkpoint_int8(step))
        torch.cuda.synchronize()
    assert torch.equal(a, step)


@pytest.mark.parametrize("m,n", [(1, 8), (40, 264), (333, 1000), (2048, 7168)])
def test_partial_sums_in_turn(m, n):
    """The bias gradient of two output gradients, through one workspace."""
    from dsv4_b200 import _native as N
    dys = [rand(m, n, seed=s, std=s) for s in (1, 3)]
    slabs = max(1, min(4 * 148 // -(-n // 256), -(-m // 32)))
    partial = torch.empty(slabs, n, device="cuda")
    outs = torch.full((TURNS, n), 7.0, dtype=BF16, device="cuda")
    st = stream()

    def call(dy, out):
        N.call("dsv4_b200_act_backward", dy.data_ptr(), n, None, 0, None, m, n, 2, 0, None, n, partial.data_ptr(), slabs,
               out.data_ptr(), st)

    want = torch.full((2, n), 7.0, dtype=BF16, device="cuda")
    for i in range(2):
        call(dys[i], want[i])
        exact = dys[i].double().sum(0)
        bound = 2.0 ** -8 * exact.abs() + (m + 8) * 2.0 ** -23 * dys[i].double().abs().sum(0) * 1.01
        assert bool(((want[i].double() - exact).abs() <= bound).all())
    for i in range(TURNS):
        call(dys[i & 1], outs[i])
    for i in range(TURNS):
        assert torch.equal(outs[i], want[i & 1]), i


@pytest.mark.parametrize("by_rows", [True, False])
@pytest.mark.parametrize("rows,cols", [(1, 7), (64, 1001), (2048, 1023)])
def test_packed_rows_in_turn(rows, cols, by_rows):
    """Rows packed twice in a row, the second time from the first's result:
    by rows of an odd stride, or by columns."""
    from dsv4_b200 import _native as N
    ld = cols + 1 if by_rows else rows + 1
    flat = [rand((rows if by_rows else cols) * ld + 1, seed=s)[1:] for s in (1, 2)]
    wide = -(-cols // 8) * 8
    first = torch.empty(rows, wide, dtype=BF16, device="cuda")
    outs = torch.full((TURNS, rows, wide + 8), math.nan, dtype=BF16, device="cuda")
    st = stream()
    strides = (ld, 1) if by_rows else (1, ld)
    want = [torch.as_strided(f, (rows, cols), strides, f.storage_offset()).contiguous() for f in flat]
    torch.cuda.synchronize()
    for i in range(TURNS):
        N.call("dsv4_b200_pack_rows", flat[i & 1].data_ptr(), *strides, rows, cols, first.data_ptr(), wide, st)
        N.call("dsv4_b200_pack_rows", first.data_ptr(), wide, 1, rows, cols, outs[i].data_ptr(), wide + 8, st)
    for i in range(TURNS):
        assert torch.equal(outs[i, :, :cols], want[i & 1]), i
        assert torch.isnan(outs[i, :, wide:]).all()
