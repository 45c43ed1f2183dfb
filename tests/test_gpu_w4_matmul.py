"""Products with 4-bit weights and group scales, and the conversion to them, against FP64 on the CPU."""
import threading

import pytest
import torch

import w4_ref as ref

pkg = ref.pkg
pytestmark = pytest.mark.gpu


def _run(codes, scales, rows, cols, group, x, pad=0, stream=None):
    """y [T][rows], written into rows `pad` elements further apart whose padding must stay as it was; the workspace starts as NaN."""
    w = ref.handle(codes, scales, rows, cols, group)
    T = x.shape[0]
    buf = torch.full((T + 1, rows + pad), 7.0, device="cuda", dtype=x.dtype)
    ws = torch.full((pkg.w4_matmul_workspace(w, x) // 4 + 64,), float("nan"), device="cuda")
    pkg.w4_matmul(w, x, buf[:T, :rows], ws, stream=stream)
    torch.cuda.synchronize()
    pkg.w4_status()
    assert bool((buf[:T, rows:] == 7.0).all()) and bool((buf[T] == 7.0).all())
    return buf[:T, :rows].cpu()


def _check(y, w, x):
    xd = x.cpu().double()
    want = xd @ w.t()
    off = ref.product_bound(w, xd, x.dtype == torch.float32) + ref.rounded(want, x.dtype)
    worst = ((y.double() - want).abs() / off).max()
    assert worst <= 1.0, float(worst)


SHAPES = [
    (1, 1, 32, 1), (1, 31, 64, 3), (15, 33, 32, 1), (17, 128, 128, 2), (16, 129, 128, 5), (130, 64, 64, 4), (100, 1000, 32, 8),
    (128, 256, 128, 16), (129, 257, 64, 17), (300, 1234, 32, 33), (257, 2050, 128, 64), (64, 4096, 64, 65), (520, 512, 128, 130),
    (1000, 700, 64, 1), (40, 12345, 128, 9), (384, 640, 32, 200), (255, 1152, 128, 257),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,group,T", SHAPES)
def test_product(gpu_lib, rows, cols, group, T, dtype):
    rng = torch.Generator().manual_seed(rows * 7919 + cols * 31 + T)
    codes, scales = ref.make(rng, rows, cols, group)
    x = torch.randn((T, cols), generator=rng).to(dtype)
    _check(_run(codes, scales, rows, cols, group, x.cuda(), pad=T % 3), ref.values(codes, scales, cols, group), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,group", [(33, 128, 32), (260, 640, 64), (144, 1100, 128), (50, 4224, 32), (300, 8192, 128), (20, 16384, 64)])
def test_small_integers_come_out_exactly(gpu_lib, rows, cols, group, dtype):
    """Integers, and scales that are powers of two: every product and sum is a number that FP32 holds, so whatever the order of additions
    the result is the integer one. |x| <= 8, |code - 8| <= 8, scales from 1 to 8 and 16384 columns: below 2^23."""
    rng = torch.Generator().manual_seed(rows)
    codes, scales = ref.make(rng, rows, cols, group)
    groups = -(-cols // group)
    scales[:, :groups] = torch.exp2(torch.randint(0, 4, (rows, groups), generator=rng).float()).to(torch.bfloat16)
    w = ref.values(codes, scales, cols, group)
    for T in (1, 2, 3, 4, 5, 16, 17, 33, 64, 65, 129):
        x = torch.randint(-8, 9, (T, cols), generator=rng).to(dtype)
        y = _run(codes, scales, rows, cols, group, x.cuda())
        want = x.double() @ w.t()
        assert torch.equal(y.double(), want.to(dtype).double()), T


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,group,T", [(40, 9728, 32, 2), (40, 9729, 128, 2), (33, 9729, 64, 1), (30, 17152, 32, 1), (30, 17153, 128, 1),
                                               (20, 27649, 64, 1), (300, 131072, 128, 1), (17, 131072, 32, 1), (20, 131071, 64, 3)])
def test_wide_rows(gpu_lib, rows, cols, group, T, dtype):
    """Columns on both sides of where two rows' digits no longer fit, and one row's, up to the most that there may be."""
    rng = torch.Generator().manual_seed(cols + T)
    codes, scales = ref.make(rng, rows, cols, group)
    x = torch.randn((T, cols), generator=rng).to(dtype)
    _check(_run(codes, scales, rows, cols, group, x.cuda(), pad=T % 3), ref.values(codes, scales, cols, group), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,group,T", [(9473, 100, 32, 1), (9500, 2048, 128, 2), (20011, 1050, 64, 4), (12288, 1920, 32, 3), (9999, 129, 128, 1)])
def test_many_short_rows(gpu_lib, rows, cols, group, T, dtype):
    rng = torch.Generator().manual_seed(rows + T)
    codes, scales = ref.make(rng, rows, cols, group)
    x = torch.randn((T, cols), generator=rng).to(dtype)
    _check(_run(codes, scales, rows, cols, group, x.cuda(), pad=T % 3), ref.values(codes, scales, cols, group), x)



@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 4, 30, 100])
def test_small_columns_beside_large_ones(gpu_lib, T, dtype):
    """The first 128 columns of x are 2^24 times the others and have zero weights. What many rows are held to is 2^-38 of the row's
    largest then (half a step of 2^-24 beside at least 2^13), which is above 2^-22 of the others."""
    rows, cols, group = 50, 384, 64
    rng = torch.Generator().manual_seed(T)
    codes, scales = ref.make(rng, rows, cols, group)
    codes[:, :64] = 0x88
    x = torch.randn((T, cols), generator=rng)
    x[:, :128] *= 2.0 ** 24
    x = x.to(dtype)
    w, xd = ref.values(codes, scales, cols, group), x.double()
    y, want = _run(codes, scales, rows, cols, group, x.cuda()).double(), xd @ w.t()
    off = ref.product_bound(w, xd, dtype == torch.float32) + ref.rounded(want, dtype) + 2.0 ** -38 * xd.abs().amax(1)[:, None] * w.abs().sum(1)
    assert bool(((y - want).abs() <= off).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 40])
def test_columns_far_above_their_neighbours(gpu_lib, T, group, dtype):
    """In each 128 columns two, an even and an odd one, are 2^13 times the others and have zero weights: what their neighbours are off must not
    show in the product. An activation is held to 2^-29 of the largest of its 128 columns in calls of one or two rows, else to 2^-22 of
    itself (BF16: exactly) and 2^-38 of its row's largest; that few numbers are added makes the sums' own share small."""
    rows, cols = 300, 256
    rng = torch.Generator().manual_seed(T + group)
    codes, scales = ref.make(rng, rows, cols, group)
    x = torch.randn((T, cols), generator=rng)
    for c in (18, 77, 128 + 1, 128 + 126):
        x[:, c] = 2.0 ** 13 * (1.0 + torch.rand(T, generator=rng))
        at = codes[:, c // 2]
        codes[:, c // 2] = (at & 15) | 0x80 if c % 2 else (at & 0xf0) | 8
    x = x.to(dtype)
    w, xd = ref.values(codes, scales, cols, group), x.double()
    y, want = _run(codes, scales, rows, cols, group, x.cuda()).double(), xd @ w.t()
    steps = 2 * (cols // 16 + 1) + cols // 32 + 16
    block = xd.abs().view(T, -1, 128).amax(2).repeat_interleave(128, 1)
    off = (xd.abs() @ w.abs().t()) * (steps * 2.0 ** -23 + (2.0 ** -22 if dtype == torch.float32 else 0.0))
    off = off + (block * 2.0 ** -29 + xd.abs().amax(1, keepdim=True) * 2.0 ** -38) @ w.abs().t() + ref.rounded(want, dtype)
    assert bool(((y - want).abs() <= off).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64])
@pytest.mark.parametrize("T", [1, 4, 30, 100])
def test_scales_far_apart(gpu_lib, T, group, dtype):
    """Neighbouring groups' scales from 1 down to 2^-12 (exact), 2^-27 (exact), or 2^-40 of each other, the large ones' weights zero: 2^-36 of
    the largest scale (half a step of F16's 2^-24 beside 2^11 at least) is what a product may then be off in many rows."""
    rows, cols = 96, 256
    rng = torch.Generator().manual_seed(T + group)
    codes, scales = ref.make(rng, rows, cols, group)
    at = torch.arange(cols // group) % 2 == 1
    ratio = 2.0 ** -torch.tensor([12.0, 27.0, 40.0])[torch.arange(rows) % 3]
    scales[:, :cols // group] = torch.where(at[None], ratio[:, None].expand(rows, cols // group), torch.ones(rows, cols // group)).to(torch.bfloat16)
    codes.view(rows, cols // group, group // 2)[:, ~at] = 0x88
    x = torch.randn((T, cols), generator=rng).to(dtype)
    w, xd = ref.values(codes, scales, cols, group), x.double()
    y, want = _run(codes, scales, rows, cols, group, x.cuda()).double(), xd @ w.t()
    off = ref.product_bound(w, xd, dtype == torch.float32) + ref.rounded(want, dtype)
    off[:, 2::3] += 2.0 ** -36 * xd.abs().sum(1)[:, None]
    assert bool(((y - want).abs() <= off).all())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 3, 40, 70])
def test_low_bits_beside_a_large_sum(gpu_lib, T, group):
    """2^17 and then 7 times 16 columns of 32 + 29 2^-15, all weights one. In F16 terms the upper ones are multiples of the sum's unit, 2^-6, the lower ones of
    16 columns 0.9 of it: a matrix instruction that adds those to the sum cuts them off, 6.3 units in all. Added up before the large ones they are cut
    once, by less than a unit for each of an instruction's two cuts."""
    rows, cols = 70, 128
    codes, scales = ref.make(torch.Generator().manual_seed(1), rows, cols, group)
    codes[:] = 0x99
    scales[:, :cols // group] = 1.0
    x = torch.full((T, cols), 32.0 + 29 * 2.0 ** -15)
    x[:, :16] = 2.0 ** 13
    y = _run(codes, scales, rows, cols, group, x.cuda()).double()
    assert bool(((y - x[0].double().sum()).abs() <= 2 * 2.0 ** -6).all())


@pytest.mark.parametrize("T", [1, 4, 30, 100])
def test_zero_weights_give_zero(gpu_lib, T):
    rows, cols, group = 70, 500, 32
    codes, scales = ref.make(torch.Generator().manual_seed(1), rows, cols, group)
    codes[:] = 0x88
    codes[3, 7] = 0x98                                      # one weight (row 3, column 15) that is not
    x = torch.randn((T, cols), generator=torch.Generator().manual_seed(2)) * 1e3
    y = _run(codes, scales, rows, cols, group, x.cuda())
    keep = torch.arange(rows) != 3
    assert bool((y[:, keep] == 0).all())
    _check(y, ref.values(codes, scales, cols, group), x)


def test_no_rows(gpu_lib):
    codes, scales = ref.make(torch.Generator().manual_seed(1), 8, 64, 32)
    y = _run(codes, scales, 8, 64, 32, torch.zeros((0, 64), device="cuda"))
    assert y.shape == (0, 8)


@pytest.mark.parametrize("T", [1, 20])
def test_matrix_over_four_gigabytes(gpu_lib, T):
    """Rows on both sides of 2^31 and 2^32 bytes of codes, and the last ones."""
    rows, cols, group = (1 << 20) + 4101, 8448, 128
    pitch, sp = pkg.w4_pitch(cols), pkg.w4_scale_pitch(cols, group)
    codes = torch.full((rows, pitch), 0x88, dtype=torch.uint8, device="cuda")
    scales = torch.ones((rows, sp), dtype=torch.bfloat16, device="cuda")
    rng = torch.Generator().manual_seed(9)
    at = sorted({0, 1, (1 << 31) // pitch, (1 << 31) // pitch + 1, (1 << 32) // pitch, (1 << 32) // pitch + 1, rows - 2, rows - 1})
    some = torch.randint(0, 256, (len(at), pitch), generator=rng, dtype=torch.int32).to(torch.uint8)
    codes[at] = some.cuda()
    x = torch.randint(-4, 5, (T, cols), generator=rng).float()
    w = pkg.W4(codes, scales, rows, cols, group)
    y = torch.empty((T, rows), device="cuda")
    ws = torch.empty(pkg.w4_matmul_workspace(w, x.cuda()), dtype=torch.uint8, device="cuda")
    pkg.w4_matmul(w, x.cuda(), y, ws)
    pkg.w4_status()
    want = x.double() @ ref.values(some, torch.ones((len(at), sp), dtype=torch.bfloat16), cols, group).t()
    assert torch.equal(y[:, at].cpu().double(), want)
    y[:, at] = 0
    assert int(y.count_nonzero()) == 0


@pytest.mark.parametrize("T", [1, 7, 40, 150])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_apart_and_off_every_alignment(gpu_lib, dtype, T):
    rng = torch.Generator().manual_seed(T)
    rows, cols, group = 77, 261, 64
    codes, scales = ref.make(rng, rows, cols, group)
    whole = torch.randn((T, cols + 10), generator=rng).to(dtype)
    on = whole.cuda()
    for first in (1, 2, 8):
        y = _run(codes, scales, rows, cols, group, on[:, first:first + cols], pad=5)
        _check(y, ref.values(codes, scales, cols, group), whole[:, first:first + cols])


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("T", [2, 100])
def test_magnitudes_far_apart(gpu_lib, T, group):
    """Rows of x from 2^-120 to 2^60, values of a row over 2^30, scales of a row of W over 2^40."""
    rng = torch.Generator().manual_seed(3 + T)
    rows, cols = 130, 640
    codes, scales = ref.make(rng, rows, cols, group, spread=6.0)
    x = torch.randn((T, cols), generator=rng) * torch.exp2(torch.randint(-30, 1, (T, cols), generator=rng).float())
    x = x * torch.exp2(torch.linspace(-120, 60, T))[:, None]
    _check(_run(codes, scales, rows, cols, group, x.cuda()), ref.values(codes, scales, cols, group), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 2, 5, 40, 70])
def test_scales_and_activations_of_every_magnitude(gpu_lib, T, group, dtype):
    """Rows of W with scales from 2^-125 to 2^124, rows of x from 2^-120 to 2^120: wherever the magnitudes of a result's products add up to less
    than the largest number, it is as exact as others, but for what falls below FP32's range: 2^-127 of the activations, and 2^-126."""
    rows, cols = 96, 640
    rng = torch.Generator().manual_seed(T + group)
    codes, scales = ref.make(rng, rows, cols, group, scale=1.0)
    groups = cols // group
    k = torch.tensor([-125, -100, -50, 0, 50, 90, 110, 124])[torch.arange(rows) % 8]
    scales[:, :groups] = (scales[:, :groups].double().clamp(max=8.0) * torch.exp2(k.double())[:, None]).to(torch.bfloat16)
    assert bool(torch.isfinite(scales[:, :groups]).all())
    w = ref.values(codes, scales, cols, group)
    seen = 0
    for j in (-120, -90, -40, 0, 30, 70, 105, 120):
        x = (torch.randn((T, cols), generator=rng).double() * torch.exp2(j + 4.0 * (torch.arange(T) % 2).double())[:, None]).to(dtype)
        xd = x.double()
        y, want, sums = _run(codes, scales, rows, cols, group, x.cuda()).double(), xd @ w.t(), xd.abs() @ w.abs().t()
        off = ref.product_bound(w, xd, dtype == torch.float32) + ref.rounded(want, dtype) + 2.0 ** -127 * xd.abs().sum(1, keepdim=True)
        inside = sums < 2.0 ** 127.9
        seen += int(inside.sum())
        assert bool(((y - want).abs() <= off)[inside].all())
    assert seen > 3 * T * rows


@pytest.mark.parametrize("T", [1, 5, 90])
def test_rows_without_numbers(gpu_lib, T):
    """A row of zeros is zero; one with an infinity or NaN is NaN in all outputs; its neighbours do not see it."""
    rng = torch.Generator().manual_seed(5)
    rows, cols, group = 200, 300, 128
    codes, scales = ref.make(rng, rows, cols, group)
    w = ref.values(codes, scales, cols, group)
    for what in (0.0, float("inf"), float("-inf"), float("nan")):
        x = torch.randn((T, cols), generator=rng)
        bad = T // 2
        if what == 0.0:
            x[bad] = 0.0
        else:
            x[bad, 17] = what
        y = _run(codes, scales, rows, cols, group, x.cuda())
        assert bool((y[bad] == 0.0).all()) if what == 0.0 else bool(torch.isnan(y[bad]).all())
        keep = torch.arange(T) != bad
        if bool(keep.any()):
            _check(y[keep], w, x[keep])


@pytest.mark.parametrize("T", [1, 6, 70])
def test_same_bits_every_time_on_any_stream_and_in_a_graph(gpu_lib, T):
    rng = torch.Generator().manual_seed(11)
    rows, cols, group = 1000, 2048, 128
    codes, scales = ref.make(rng, rows, cols, group)
    x = torch.randn((T, cols), generator=rng).cuda()
    first, second = _run(codes, scales, rows, cols, group, x), _run(codes, scales, rows, cols, group, -x)
    side = torch.cuda.Stream()
    assert torch.equal(_run(codes, scales, rows, cols, group, x, stream=side.cuda_stream), first)
    # two captured calls with workspaces of their own, replayed beside each other with new inputs
    w = ref.handle(codes, scales, rows, cols, group)
    graphs, ins, outs, spaces = [], [], [], []
    torch.cuda.synchronize()
    for i in range(2):
        ins.append(torch.zeros_like(x))
        outs.append(torch.zeros((T, rows), device="cuda"))
        spaces.append(torch.empty(pkg.w4_matmul_workspace(w, x), dtype=torch.uint8, device="cuda"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            pkg.w4_matmul(w, ins[i], outs[i], spaces[i])
        graphs.append(g)
    ins[0].copy_(x)
    ins[1].copy_(-x)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0].cpu(), first) and torch.equal(outs[1].cpu(), second)


@pytest.mark.parametrize("T", [1, 2, 5, 70])
def test_refused_calls_write_nothing(gpu_lib, T):
    """A workspace a byte short or off its alignment, a matrix or a row on the host: an error that says so, and y stays as it was."""
    rows, cols, group = 40, 96, 32
    codes, scales = ref.make(torch.Generator().manual_seed(T), rows, cols, group)
    w = ref.handle(codes, scales, rows, cols, group)
    x, y = torch.ones((T, cols), device="cuda"), torch.full((T, rows), 3.0, device="cuda")
    need = pkg.w4_matmul_workspace(w, x)
    space = torch.empty(need + 512, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError, match=f"has {need - 1} bytes, {need} are needed"):
        pkg.w4_matmul(w, x, y, space[:need - 1])
    with pytest.raises(RuntimeError, match="workspace must lie on a multiple of 256 bytes"):
        pkg.w4_matmul(w, x, y, space[16:])
    with pytest.raises(RuntimeError, match="the matrix is not device memory"):
        pkg._call_w4("g5b_w4_matmul", pkg.W4(codes, scales, rows, cols, group).ref, x.data_ptr(), 0, T, cols, y.data_ptr(), rows, space.data_ptr(), need, 0)
    with pytest.raises(RuntimeError, match="x is not device memory"):
        pkg._call_w4("g5b_w4_matmul", w.ref, x.cpu().data_ptr(), 0, T, cols, y.data_ptr(), rows, space.data_ptr(), need, 0)
    torch.cuda.synchronize()
    assert bool((y == 3.0).all())
    pkg.w4_matmul(w, x, y, space[:need])
    _check(y.cpu(), ref.values(codes, scales, cols, group), x)


def test_threads_of_their_own(gpu_lib):
    """Threads that call at once, each on a stream and with a workspace of its own, with products that want more shared memory one after the other:
    what one thread alone gets, bit for bit."""
    rng = torch.Generator().manual_seed(3)
    work = []
    for rows, cols, group in ((200, 320, 32), (300, 4096, 128), (100, 9000, 64)):
        codes, scales = ref.make(rng, rows, cols, group)
        for T in (1, 2, 5, 70):
            work.append((ref.handle(codes, scales, rows, cols, group), torch.randn((T, cols), generator=rng).cuda()))

    def run(order, out):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for i in order:
                w, x = work[i]
                y = torch.empty((x.shape[0], w.rows), device="cuda")
                pkg.w4_matmul(w, x, y, torch.empty(pkg.w4_matmul_workspace(w, x), dtype=torch.uint8, device="cuda"))
                out[i] = y
        stream.synchronize()

    torch.cuda.synchronize()
    got = [{} for _ in range(6)]
    threads = [threading.Thread(target=run, args=([(i * step + k) % len(work) for i in range(len(work))], got[k])) for k, step in enumerate((1, 5, 7, 11, 1, 5))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    alone = {}
    run(range(len(work)), alone)
    pkg.w4_status()
    for out in got:
        assert len(out) == len(work) and all(torch.equal(out[i], alone[i]) for i in alone)


def test_status_waits_for_the_current_stream(gpu_lib):
    """A product behind some milliseconds of work on a side stream: the look, which is given no stream, comes after it."""
    rows, cols, group = 300, 512, 128
    codes, scales = ref.make(torch.Generator().manual_seed(1), rows, cols, group)
    w, x, y = ref.handle(codes, scales, rows, cols, group), torch.ones((40, cols), device="cuda"), torch.empty((40, rows), device="cuda")
    space = torch.empty(pkg.w4_matmul_workspace(w, x), dtype=torch.uint8, device="cuda")
    big = torch.ones((8192, 8192), device="cuda", dtype=torch.bfloat16)
    side, out = torch.cuda.Stream(), torch.empty_like(big)
    for n in (1, 40):                                      # (what is set up at a first use waits for the device)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(n):
                torch.mm(big, big, out=out)
            pkg.w4_matmul(w, x, y, space)
            pkg.w4_status()
            assert side.query()
    _check(y.cpu(), ref.values(codes, scales, cols, group), x)


# ------------------------------------------------------------------ conversion ----
def _quantized(v, group):
    """(codes as numbers 0..15 [rows][cols], scales [rows][groups]) of FP32 values, quotients in FP64."""
    rows, cols = v.shape
    groups = -(-cols // group)
    p = torch.nn.functional.pad(v.double(), (0, groups * group - cols)).view(rows, groups, group)
    m = p.abs().amax(2)
    s = (m / 7.0).float().to(torch.bfloat16)
    s = torch.where(torch.isfinite(m), s, torch.tensor(float("nan"), dtype=torch.bfloat16))
    q = (p / s.double()[..., None]).round().clamp(-7, 7)
    q = torch.where((s.double()[..., None] > 0) & torch.isfinite(q), q, 0.0)
    return (q + 8).to(torch.uint8).view(rows, -1)[:, :cols], s


def _convert(src, rows, cols, group, scale=None, block=(128, 128)):
    codes = torch.full((rows, pkg.w4_pitch(cols)), 255, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows, pkg.w4_scale_pitch(cols, group)), float("nan"), dtype=torch.bfloat16, device="cuda")
    w = pkg.W4(codes, scales, rows, cols, group)
    pkg.w4_quantize(src.cuda(), w, scale_inv=scale.cuda() if scale is not None else None, block=block)
    out = {}
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.full((rows, cols + 3), 5.0, device="cuda", dtype=dt)
        pkg.w4_dequantize(w, buf[:, :cols])
        torch.cuda.synchronize()
        assert bool((buf[:, cols:] == 5.0).all())
        out[dt] = buf[:, :cols].cpu()
    return codes.cpu(), scales.cpu(), out


def _compare(v, got, rows, cols, group):
    codes, scales, out = got
    want, s = _quantized(v, group)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    assert torch.equal(c[:, :cols], want)
    assert bool((c[:, cols:] == 8).all()) and bool((scales[:, s.shape[1]:] == 0).all())
    assert torch.equal(scales[:, :s.shape[1]].view(torch.int16)[~torch.isnan(s)], s.view(torch.int16)[~torch.isnan(s)])
    assert torch.equal(torch.isnan(scales[:, :s.shape[1]]), torch.isnan(s))
    y = (want.double() - 8) * s.double().repeat_interleave(group, 1)[:, :cols]
    for dt, o in out.items():
        assert torch.equal(torch.nan_to_num(o, nan=123.0), torch.nan_to_num(y.to(dt), nan=123.0))


@pytest.mark.parametrize("rows,cols,group", [(1, 1, 32), (3, 33, 32), (5, 64, 64), (7, 200, 128), (64, 1024, 32), (33, 1031, 64), (9, 5000, 128), (2, 4097, 32)])
@pytest.mark.parametrize("kind", ["f32", "bf16", "fp8"])
def test_quantize_and_back(gpu_lib, rows, cols, group, kind):
    rng = torch.Generator().manual_seed(rows + cols)
    v, scale = 0.02 * torch.randn((rows, cols), generator=rng), None
    if kind == "bf16":
        src = v.to(torch.bfloat16)
        v = src.float()
    elif kind == "fp8":
        for block in ((128, 128), (16, 12)):
            scale = 1e-4 * (1 + torch.rand((-(-rows // block[0]), -(-cols // block[1])), generator=rng))
            src = (v * 5000).to(torch.float8_e4m3fn)
            vv = src.float() * scale.repeat_interleave(block[0], 0)[:rows].repeat_interleave(block[1], 1)[:, :cols]
            _compare(vv, _convert(src, rows, cols, group, scale, block), rows, cols, group)
        return
    else:
        src = v
    _compare(v, _convert(src, rows, cols, group), rows, cols, group)


@pytest.mark.parametrize("kind,shifts", [("f32", (0, 1, 2, 3)), ("bf16", (0, 1, 3, 7)), ("fp8", (0, 1, 2, 3, 5))])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 3), (5, 31), (4, 1023), (3, 1025), (6, 2049), (37, 1282), (2, 4100),
                                       (130, 20), (70, 100), (33, 128), (37, 161), (9, 256), (17, 504), (33, 511), (19, 512), (5, 513)])
def test_quantize_rows_that_lie_anyhow(gpu_lib, rows, cols, kind, shifts):
    """Sources from any element on, beside numbers that would show (NaN); F32 and BF16 values back into rows of any distance."""
    rng = torch.Generator().manual_seed(rows + cols)
    v, scale = 0.02 * torch.randn((rows, cols), generator=rng), None
    if kind == "bf16":
        v = v.to(torch.bfloat16)
    elif kind == "fp8":
        scale = 1e-4 * (1 + torch.rand((-(-rows // 16), -(-cols // 12)), generator=rng))
        v = (v * 5000).to(torch.float8_e4m3fn)
    for shift in shifts:
        buf = torch.full((rows * cols + 16,), float("nan"), device="cuda").to(v.dtype)
        src = buf[shift:shift + rows * cols].view(rows, cols)
        src.copy_(v)
        vv = v.float() * scale.repeat_interleave(16, 0)[:rows].repeat_interleave(12, 1)[:, :cols] if kind == "fp8" else v.float()
        group = (32, 64, 128)[shift % 3]
        _compare(vv, _convert(src, rows, cols, group, scale, (16, 12)), rows, cols, group)


def test_quantize_borders(gpu_lib):
    """Quotients at, and one FP32 step to either side of, every half; groups of zeros, of subnormal and of huge values, and without numbers."""
    group, rows = 32, 64
    v = torch.zeros((rows, 5 * group))
    for r in range(rows):
        top = (1.0 + r / 64.0) * 2.0 ** (r % 7 - 20)
        s = (torch.tensor(top, dtype=torch.float64) / 7).float().to(torch.bfloat16).double()
        half = torch.tensor([(k + 0.5) * float(s) for k in range(-7, 7)], dtype=torch.float32)
        inf = torch.tensor(float("inf"))
        v[r, 0], v[r, group], v[r, 2 * group] = top, -top, top
        v[r, 1:15] = half
        v[r, group + 1:group + 15] = torch.nextafter(half, inf)
        v[r, 2 * group + 1:2 * group + 15] = torch.nextafter(half, -inf)
        v[r, 4 * group:] = torch.linspace(-1, 1, group) * 2.0 ** (-149 + 2 * r if r < 40 else 127 - (r - 40))
    v[5, 3 * group + 3], v[6, 3 * group + 31], v[7, 3 * group] = float("nan"), float("inf"), float("-inf")
    _compare(v, _convert(v, rows, 5 * group, group), rows, 5 * group, group)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("exponent", [-130, -101, -20, 100])
def test_quantize_every_quotient_of_bf16(gpu_lib, kind, exponent):
    """Every BF16 number from a 64th of a scale on, of both signs, beside every significand of the largest (and so all of the scale's):
    exact halves and what lies nearest to them."""
    group = 128
    top = (128 + torch.arange(128)).double() * 2.0 ** (exponent - 7)
    others = torch.cat([(128 + torch.arange(128)).double() * 2.0 ** (exponent - 7 - d) for d in range(9)])
    others = torch.cat((others, -others))
    others = torch.nn.functional.pad(others, (0, -len(others) % (group - 1))).view(-1, group - 1)
    rows, groups = len(top), len(others)
    v = torch.cat((top[:, None, None].expand(rows, groups, 1), others.expand(rows, groups, group - 1)), 2)
    v = torch.where(v.abs() <= top[:, None, None], v, torch.zeros(())).view(rows, groups * group).to(torch.bfloat16)
    _compare(v.float(), _convert(v if kind == "bf16" else v.float(), rows, groups * group, group), rows, groups * group, group)
