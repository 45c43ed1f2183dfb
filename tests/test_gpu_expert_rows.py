"""Tokens sorted by expert and back, and routed experts with 4-bit weights, against plain forms."""
import pytest
import torch

import w4_ref as ref

pkg = ref.pkg
pytestmark = pytest.mark.gpu


def _sorted(idx, E):
    """(order, place, offsets) by definition."""
    T, K = idx.shape
    flat = idx.flatten().tolist()
    by = sorted((p for p, e in enumerate(flat) if 0 <= e < E), key=lambda p: flat[p])
    place = [-1] * (T * K)
    for i, p in enumerate(by):
        place[p] = i
    offsets = [sum(1 for p in by if flat[p] < e) for e in range(E + 1)] if T * K < 3000 else torch.bincount(
        torch.tensor([flat[p] for p in by], dtype=torch.int64), minlength=E).cumsum(0).tolist()
    if len(offsets) == E:
        offsets = [0] + offsets
    t = lambda v: torch.tensor(v, dtype=torch.int32)        # noqa: E731
    return t(by + [-1] * (T * K - len(by))), t(place).view(T, K), t(offsets)


def _sort(idx, E):
    T, K = idx.shape
    out = [torch.full(s, 77, dtype=torch.int32, device="cuda") for s in ((T * K,), (T, K), (E + 1,))]
    pkg.expert_sort(idx.cuda(), E, *out)
    return out


def _picks(rng, T, K, E, how):
    if how == "one":
        return torch.full((T, K), E - 1, dtype=torch.int32)
    if how == "none":
        return torch.full((T, K), -1, dtype=torch.int32)
    if how == "outside":          # half of them other ranks', on both sides
        return torch.randint(-E // 2 - 1, E + E // 2 + 1, (T, K), generator=rng, dtype=torch.int32)
    if how == "elsewhere":        # seven of eight
        return torch.randint(0, 8 * E, (T, K), generator=rng, dtype=torch.int32)
    if how == "skewed":
        return (E * torch.rand((T, K), generator=rng) ** 4).to(torch.int32).clamp(max=E - 1)
    return torch.randint(0, E, (T, K), generator=rng, dtype=torch.int32)


@pytest.mark.parametrize("T,K,E", [(1, 1, 1), (1, 8, 288), (3, 5, 7), (64, 8, 288), (512, 8, 36), (513, 8, 36), (700, 6, 1024), (4097, 8, 288), (9000, 4, 3)])
@pytest.mark.parametrize("how", ["even", "skewed", "outside", "one", "none"])
def test_sort(gpu_lib, T, K, E, how):
    idx = _picks(torch.Generator().manual_seed(T + E), T, K, E, how)
    for got, want in zip(_sort(idx, E), _sorted(idx, E)):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,E,cols,pad,how", [(1, 8, 288, 4096, 0, "even"), (5, 3, 4, 1, 0, "outside"), (37, 8, 36, 255, 1, "outside"),
                                                (64, 2, 9, 1000, 8, "skewed"), (600, 8, 36, 72, 0, "outside"), (9, 4, 5, 33, 7, "none")])
def test_gather_and_combine(gpu_lib, T, K, E, cols, pad, how, dtype):
    rng = torch.Generator().manual_seed(T * cols)
    idx = _picks(rng, T, K, E, how)
    x = torch.randn((T, cols), generator=rng).to(dtype)
    weights = torch.rand((T, K), generator=rng)
    order, place, offsets = _sort(idx, E)
    wide = torch.full((T, cols + pad), 3.0, dtype=dtype)
    wide[:, :cols] = x
    rows = torch.full((T * K, cols + pad), 9.0, device="cuda", dtype=dtype)
    pkg.expert_gather(wide.cuda()[:, :cols], order, offsets, rows[:, :cols])
    n = int(offsets[-1])
    got = rows.cpu()
    assert torch.equal(got[:n, :cols], x[order[:n].cpu().long() // K])
    assert bool((got[n:] == 9.0).all()) and bool((got[:, cols:] == 9.0).all())
    # rows of their own for every pick, so that a wrong place shows
    rows[:n, :cols] = torch.randn((n, cols), generator=rng).to(dtype).cuda()
    for w in (weights, None):
        out = torch.full((T, cols + pad), 2.0, device="cuda", dtype=dtype)
        pkg.expert_combine(rows[:, :cols], place, w.cuda() if w is not None else None, out[:, :cols])
        took = rows.cpu().double()[:, :cols][place.cpu().clamp(min=0).long()] * (place.cpu() >= 0)[..., None]
        part = took * (w.double() if w is not None else torch.ones(T, K, dtype=torch.float64))[..., None]
        want = part.sum(1)
        off = part.abs().sum(1) * K * 2.0 ** -24 + ref.rounded(want, dtype)      # K fused steps, each rounded to half of 2^-23
        assert bool(((out.cpu()[:, :cols].double() - want).abs() <= off).all())
        assert bool((out.cpu()[:, cols:] == 2.0).all())


def test_numbers_far_outside(gpu_lib):
    """The smallest and largest integers are nobody's experts; orders and places that no sort wrote are left out."""
    big, small = 2 ** 31 - 1, -2 ** 31
    idx = torch.tensor([[big, 0], [small, -1], [1, 2]], dtype=torch.int32)
    for got, want in zip(_sort(idx, 2), _sorted(idx, 2)):
        assert torch.equal(got.cpu(), want)
    x = torch.arange(3 * 8, dtype=torch.float32).view(3, 8).cuda()
    rows = torch.full((6, 8), 5.0, device="cuda")
    t = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")       # noqa: E731
    pkg.expert_gather(x, t(4, big, small, 6, -1, 0), t(0, 100), rows)
    assert torch.equal(rows[0], x[2]) and torch.equal(rows[5], x[0]) and bool((rows[1:5] == 5.0).all())
    out = torch.full((3, 8), 9.0, device="cuda")
    pkg.expert_combine(rows, t(0, big, small, 6, 5, -7).view(3, 2), None, out)
    assert torch.equal(out[0], rows[0]) and bool((out[1] == 0).all()) and torch.equal(out[2], rows[5])


@pytest.mark.parametrize("K", [1, 64])
def test_no_tokens_and_many_picks(gpu_lib, K):
    E = 3
    none = torch.zeros((0, K), dtype=torch.int32)
    order, place, offsets = _sort(none, E)
    assert offsets.cpu().tolist() == [0] * (E + 1)
    idx = _picks(torch.Generator().manual_seed(K), 5, K, E, "outside")
    order, place, offsets = _sort(idx, E)
    x = torch.randn((5, 40), generator=torch.Generator().manual_seed(1)).cuda()
    rows = torch.zeros((5 * K, 40), device="cuda")
    pkg.expert_gather(x, order, offsets, rows)
    out = torch.empty_like(x)
    pkg.expert_combine(rows, place, None, out)
    here = ((idx >= 0) & (idx < E)).sum(1).double()
    # every pick of a token has the token's own row: K sums, each off by half of 2^-23 of at most the whole
    want = x.cpu().double() * here[:, None]
    assert bool(((out.cpu().double() - want).abs() <= want.abs() * K * 2.0 ** -24).all())


def test_combine_does_not_read_rows_left_out(gpu_lib):
    """NaN in the rows of picks that are not here, and weights that are not numbers beside them, reach nothing."""
    idx = torch.tensor([[0, -1, 2], [5, 9, -7]], dtype=torch.int32)
    order, place, offsets = _sort(idx, 4)
    rows = torch.full((6, 8), float("nan"), device="cuda")
    rows[:2] = 1.5
    weights = torch.tensor([[2.0, float("nan"), 1.0], [float("inf")] * 3]).cuda()
    out = torch.empty((2, 8), device="cuda")
    pkg.expert_combine(rows, place, weights, out)
    assert bool((out[0] == 4.5).all()) and bool((out[1] == 0.0).all())


def _stack(rng, E, rows, cols, group):
    codes, scales = ref.make(rng, rows, cols, group, E, scale=0.03)
    return pkg.W4(codes.cuda(), scales.cuda(), rows, cols, group), ref.values(codes, scales, cols, group)


def _experts(handles, x, idx, weights, limit, pad=0):
    T, H = x.shape
    ws = torch.full((pkg.w4_experts_workspace(*handles, x, idx) // 4,), float("nan"), device="cuda")
    out = torch.full((T, H + pad), 6.0, device="cuda", dtype=x.dtype)
    pkg.w4_experts(*handles, x, idx.cuda(), weights.cuda(), limit, out[:, :H], ws)
    torch.cuda.synchronize()
    pkg.w4_status()
    assert bool((out[:, H:] == 6.0).all())
    return out[:, :H].cpu()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,E,H,I,group,limit,how", [
    (1, 8, 12, 256, 128, 128, 10.0, "even"), (1, 1, 1, 33, 17, 32, 1.0, "even"), (5, 4, 6, 200, 96, 64, float("inf"), "outside"),
    (40, 3, 4, 130, 257, 32, 0.5, "skewed"), (90, 2, 3, 384, 128, 128, 2.0, "even"), (70, 2, 5, 100, 300, 64, 10.0, "one"),
    (3, 2, 4, 64, 64, 32, 10.0, "none"), (33, 4, 40, 160, 160, 32, 3.0, "outside"),
    (16, 4, 64, 256, 130, 32, 10.0, "even"), (2, 8, 20, 700, 130, 64, 10.0, "skewed"),
    (4, 8, 256, 64, 48, 32, 10.0, "even"), (4, 8, 256, 72, 48, 32, 10.0, "outside"), (3, 8, 256, 64, 48, 32, 10.0, "none"),
    (60, 4, 40, 130, 96, 64, 10.0, "even"), (70, 8, 40, 130, 96, 32, 10.0, "elsewhere"), (100, 4, 40, 96, 130, 128, 10.0, "elsewhere"),
    (78, 8, 40, 64, 64, 64, 10.0, "elsewhere"), (90, 8, 40, 64, 64, 64, 10.0, "none")])
def test_experts(gpu_lib, T, K, E, H, I, group, limit, how, dtype):
    rng = torch.Generator().manual_seed(T * 13 + H)
    (gate, g), (up, u), (down, d) = _stack(rng, E, I, H, group), _stack(rng, E, I, H, group), _stack(rng, E, H, I, group)
    idx = _picks(rng, T, K, E, how)                        # the same expert twice in a token among them
    weights = torch.rand((T, K), generator=rng) * 2 - 0.5
    x = torch.randn((T, H), generator=rng).to(dtype)
    got = _experts((gate, up, down), x.cuda(), idx, weights, limit, pad=T % 2)
    want, off = ref.experts(x.double(), idx, weights, g, u, d, limit, dtype == torch.float32)
    worst = ((got.double() - want).abs() / (off + ref.rounded(want, dtype))).max()
    assert worst <= 1.0, float(worst)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,E,H,I,group,down_group,how", [
    (2, 2, 3, 4096, 40, 128, 64, "even"), (9, 4, 20, 4096, 24, 32, 128, "even"), (20, 4, 8, 4096, 24, 128, 32, "elsewhere"), (20, 4, 8, 4096, 24, 128, 64, "even"),
    (40, 1, 2, 4224, 40, 64, 32, "even"), (3, 2, 3, 5000, 33, 128, 32, "skewed"), (9, 4, 20, 5000, 24, 64, 64, "outside"),
    (3, 2, 3, 9728, 24, 64, 128, "even"), (9, 4, 20, 9728, 24, 128, 64, "skewed"), (3, 2, 3, 9856, 40, 32, 128, "even"), (20, 2, 3, 9856, 24, 128, 32, "even"),
    (2, 2, 3, 17280, 24, 64, 128, "even"), (2, 2, 3, 48, 4224, 64, 128, "even"), (9, 4, 20, 40, 9856, 32, 64, "even"), (3, 2, 3, 40, 9856, 128, 32, "even")])
def test_wide_experts(gpu_lib, T, K, E, H, I, group, down_group, how, dtype):
    """A piece of 4096 columns, one and a part of the next, several; the widest that two rows' digits fit beside (9728 columns), one row's, none's; the
    down matrix in groups of another size. Few experts and channels, the released width."""
    rng = torch.Generator().manual_seed(T * 7 + H + I)
    (gate, g), (up, u), (down, d) = _stack(rng, E, I, H, group), _stack(rng, E, I, H, group), _stack(rng, E, H, I, down_group)
    idx = _picks(rng, T, K, E, how)
    weights = torch.rand((T, K), generator=rng) * 2 - 0.5
    x = (0.2 * torch.randn((T, H), generator=rng)).to(dtype)
    got = _experts((gate, up, down), x.cuda(), idx, weights, 10.0, pad=T % 2)
    want, off = ref.experts(x.double(), idx, weights, g, u, d, 10.0, dtype == torch.float32)
    worst = ((got.double() - want).abs() / (off + ref.rounded(want, dtype))).max()
    assert worst <= 1.0, float(worst)


def test_experts_without_numbers_and_far_outside(gpu_lib):
    """A token with an infinity is NaN, its neighbours are not; picks far outside add nothing; a token without picks is zero."""
    rng = torch.Generator().manual_seed(21)
    E, H, I = 5, 96, 64
    (gate, g), (up, u), (down, d) = _stack(rng, E, I, H, 32), _stack(rng, E, I, H, 32), _stack(rng, E, H, I, 32)
    for T in (3, 12, 60):                                  # picks one by one, a few rows to an expert, many
        idx = torch.randint(0, E, (T, 2), generator=rng, dtype=torch.int32)
        idx[0] = torch.tensor([2 ** 31 - 1, -2 ** 31])
        x = torch.randn((T, H), generator=rng)
        x[1, 5] = float("inf")
        weights = torch.rand((T, 2), generator=rng)
        got = _experts((gate, up, down), x.cuda(), idx, weights, 10.0)
        assert bool((got[0] == 0).all()) and bool(torch.isnan(got[1]).all())
        want, off = ref.experts(x[2:].double(), idx[2:], weights[2:], g, u, d, 10.0, True)
        assert bool(((got[2:].double() - want).abs() <= off + ref.rounded(want, torch.float32)).all())
    none = torch.zeros((0, 2), dtype=torch.int32)
    assert _experts((gate, up, down), torch.zeros((0, H), device="cuda"), none, torch.zeros((0, 2)), 10.0).shape == (0, H)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E", [(3, 2), (18, 20), (20, 2), (40, 2)])
def test_hidden_rows_keep_what_fp32_holds(gpu_lib, T, E, dtype):
    """Integers past weights that are multiples of 2^-6: gate and up are exact, the hidden row is off by what the sigmoid (1.53 units of 2^-23) and two
    products are, and the down product by its additions and 2^-22 of a factor, in calls that take picks one by one, by two, and by 64."""
    rng = torch.Generator().manual_seed(T)
    H, I = 64, 32
    stack = lambda r, c, s: ref.make(rng, r, c, 32, E, spread=0.0, scale=s)        # noqa: E731
    made = [(stack(r, c, s), r, c) for r, c, s in ((I, H, 2.0 ** -6), (I, H, 2.0 ** -6), (H, I, 0.03))]
    handles, (g, u, d) = [ref.handle(*m, r, c, 32) for m, r, c in made], [ref.values(*m, c, 32) for m, r, c in made]
    idx = torch.randint(0, E, (T, 1), generator=rng, dtype=torch.int32)
    x = torch.randint(-8, 9, (T, H), generator=rng).to(dtype)
    got = _experts(handles, x.cuda(), idx, torch.ones((T, 1)), 10.0).double()
    at = idx[:, 0].long()
    h = ref.swiglu(torch.einsum("th,tih->ti", x.double(), g[at]), torch.einsum("th,tih->ti", x.double(), u[at]), 10.0)
    want = torch.einsum("ti,thi->th", h, d[at])
    steps = 2 * (I // 16 + 1) + I // 32 + 16
    off = torch.einsum("ti,thi->th", h.abs(), d[at].abs()) * (steps + 4 + 2) * 2.0 ** -23 + ref.rounded(want, dtype)
    assert bool(((got - want).abs() <= off).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("T,K,E", [(3, 2, 5), (9, 3, 20), (12, 2, 5), (60, 2, 5)])
def test_experts_of_huge_rows_and_small_weights(gpu_lib, T, K, E, group, dtype):
    """Some rows of x about 2^110, gate and up weights about 2^-100, and as large ones the other way round: all results are numbers."""
    rng = torch.Generator().manual_seed(T + group)
    H, I = 200, 150
    for big, small, down_ in ((110, -100, 1.0), (-100, 110, 2.0 ** 80)):
        made = [(ref.make(rng, r, c, group, E, scale=s), r, c) for r, c, s in ((I, H, 2.0 ** small), (I, H, 2.0 ** small), (H, I, down_))]
        handles, (g, u, d) = [ref.handle(*m, r, c, group) for m, r, c in made], [ref.values(*m, c, group) for m, r, c in made]
        idx = torch.randint(0, E, (T, K), generator=rng, dtype=torch.int32)
        x = (torch.randn((T, H), generator=rng) * torch.where(torch.arange(T) % 3 == 1, 1.0, 2.0 ** big)[:, None]).to(dtype)
        weights = torch.rand((T, K), generator=rng)
        got = _experts(handles, x.cuda(), idx, weights, float("inf"))
        want, off = ref.experts(x.double(), idx, weights, g, u, d, float("inf"), dtype == torch.float32)
        fine = want.abs() < 2.0 ** 120                     # (rows of ordinary size past huge weights: their products leave FP32)
        assert int(fine.sum()) >= H and bool(((got.double() - want).abs() <= off + ref.rounded(want, dtype))[fine].all())


def test_a_checkpoint_expert_layer_in_four_bits(gpu_lib):
    """As they are used together: FP8 experts converted one matrix at a time into stacks, a prompt and then single tokens through
    them; the layer put together from the sort, the gather, the products and the combination gives the same."""
    rng = torch.Generator().manual_seed(42)
    E, H, I, K, group = 4, 256, 128, 2, 64
    src = {}
    for name, r, c in (("gate", I, H), ("up", I, H), ("down", H, I)):
        codes = torch.empty((E, r, pkg.w4_pitch(c)), dtype=torch.uint8, device="cuda")
        scales = torch.empty((E, r, pkg.w4_scale_pitch(c, group)), dtype=torch.bfloat16, device="cuda")
        one = []
        for e in range(E):
            fp8 = torch.randn((r, c), generator=rng).to(torch.float8_e4m3fn).cuda()
            grid = (0.02 * (1 + torch.rand((-(-r // 128), -(-c // 128)), generator=rng))).cuda()
            one.append(pkg.W4(codes[e], scales[e], r, c, group))
            pkg.w4_quantize(fp8, one[e], scale_inv=grid)
        src[name] = (pkg.W4(codes, scales, r, c, group), one, ref.values(codes.cpu(), scales.cpu(), c, group))
    handles = [src[n][0] for n in ("gate", "up", "down")]
    for T in (50, 1, 1):
        idx = torch.randint(-1, E, (T, K), generator=rng, dtype=torch.int32)
        weights = torch.rand((T, K), generator=rng)
        x = torch.randn((T, H), generator=rng).cuda()
        got = _experts(handles, x, idx, weights, 10.0)
        want, off = ref.experts(x.cpu().double(), idx, weights, *(src[n][2] for n in ("gate", "up", "down")), 10.0, True)
        assert bool(((got.double() - want).abs() <= off + ref.rounded(want, torch.float32)).all())
        order, place, offsets = _sort(idx, E)
        rows = torch.zeros((T * K, H), device="cuda")
        pkg.expert_gather(x, order, offsets, rows)
        at = offsets.tolist()
        for e in range(E):
            part = rows[at[e]:at[e + 1]]
            h = [torch.empty((len(part), I), device="cuda") for _ in range(2)]
            ws = torch.empty(max(pkg.w4_matmul_workspace(src["gate"][1][e], part), pkg.w4_matmul_workspace(src["down"][1][e], h[0])), dtype=torch.uint8, device="cuda")
            for i, n in enumerate(("gate", "up")):
                pkg.w4_matmul(src[n][1][e], part, h[i], ws)
            act = ref.swiglu(h[0].double(), h[1].double(), 10.0).float()
            y = torch.empty_like(part)
            pkg.w4_matmul(src["down"][1][e], act, y, ws)
            rows[at[e]:at[e + 1]] = y
        out = torch.empty_like(x)
        pkg.expert_combine(rows, place, weights.cuda(), out)
        assert bool(((out.cpu().double() - want).abs() <= off + ref.rounded(want, torch.float32)).all())


def test_experts_repeat_and_replay(gpu_lib):
    rng = torch.Generator().manual_seed(8)
    E, H, I, K, T = 6, 256, 192, 3, 20
    handles = [_stack(rng, E, I, H, 64)[0], _stack(rng, E, I, H, 64)[0], _stack(rng, E, H, I, 64)[0]]
    idx = _picks(rng, T, K, E, "outside").cuda()
    weights = torch.rand((T, K), generator=rng).cuda()
    x = torch.randn((T, H), generator=rng).cuda()
    first = _experts(handles, x, idx, weights, 10.0)
    assert torch.equal(_experts(handles, x, idx, weights, 10.0), first)
    xin, iin, out = torch.zeros_like(x), torch.zeros_like(idx), torch.zeros_like(x)
    ws = torch.empty(pkg.w4_experts_workspace(*handles, x, idx), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pkg.w4_experts(*handles, xin, iin, weights, 10.0, out, ws)
    xin.copy_(x)
    iin.copy_(idx)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), first)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_replay_with_other_picks(gpu_lib, dtype):
    """One captured call, replayed with picks of which all, one in eight and none are here: each time what an eager call gives."""
    rng = torch.Generator().manual_seed(5)
    E, H, I, T, K = 40, 128, 96, 60, 4
    (gate, g), (up, u), (down, d) = _stack(rng, E, I, H, 32), _stack(rng, E, I, H, 32), _stack(rng, E, H, I, 32)
    x = torch.randn((T, H), generator=rng).to(dtype).cuda()
    weights = torch.rand((T, K), generator=rng).cuda()
    picks = [_picks(rng, T, K, E, how).cuda() for how in ("even", "elsewhere", "none", "skewed")]
    want = [_experts((gate, up, down), x, p, weights, 10.0) for p in picks]
    idx, out = picks[0].clone(), torch.zeros_like(x)
    ws = torch.empty(pkg.w4_experts_workspace(gate, up, down, x, idx), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.w4_experts(gate, up, down, x, idx, weights, 10.0, out, ws)
    for k in (0, 1, 2, 3, 1, 0):
        idx.copy_(picks[k])
        graph.replay()
        assert torch.equal(out.cpu(), want[k])
    pkg.w4_status()
