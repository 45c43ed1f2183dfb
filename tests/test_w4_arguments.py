"""What the 4-bit operators and the sort refuse, and their sizes: host logic, no GPU."""
import ctypes as C

import pytest
import torch

import synth

pkg = synth.pkg


def _err():
    return (pkg.lib().g5b_last_error() or b"").decode()


def test_pitches():
    for cols in (1, 31, 32, 33, 4096, 4097):
        assert pkg.w4_pitch(cols) == -(-cols // 32) * 16
        for group in (32, 64, 128):
            assert pkg.w4_scale_pitch(cols, group) == -(-(-(-cols // group)) // 8) * 8
    assert pkg.w4_pitch(0) == 0 and pkg.w4_scale_pitch(64, 48) == 0 and pkg.w4_scale_pitch(-3, 32) == 0


def _w4(codes, scales, rows, cols, group, count=1):
    return pkg._W4(codes, scales, rows, cols, group, count)


@pytest.mark.parametrize("rows,cols,group,count,word", [(0, 64, 32, 1, "outside"), (64, 0, 32, 1, "outside"), (1 << 23, 64, 32, 1, "outside"),
                                                        (64, 1 << 18, 32, 1, "outside"), (64, 64, 48, 1, "32, 64 or 128"), (64, 64, 0, 1, "32, 64 or 128"),
                                                        (64, 64, 32, 0, "matrices"), (64, 64, 32, 5000, "matrices"), (64, 64, 32, 2, "matrices")])
def test_matrices_out_of_range(rows, cols, group, count, word):
    m = _w4(1 << 20, 1 << 20, rows, cols, group, count)
    assert pkg.lib().g5b_w4_matmul(C.byref(m), 1 << 20, 0, 1, 1 << 20, 1 << 20, 1 << 23, 1 << 20, 1 << 30, None) == -1
    assert word in _err()
    assert pkg.lib().g5b_w4_dequantize(C.byref(m), 0, 1 << 20, 1 << 20, None) == -1 and word in _err()


def test_addresses():
    L, a = pkg.lib(), torch.zeros(1 << 16, dtype=torch.uint8)
    here = (a.data_ptr() + 255) // 256 * 256
    x = _w4(None, here, 16, 32, 32)
    assert L.g5b_w4_dequantize(C.byref(x), 0, here, 32, None) == -1 and "null" in _err()
    x = _w4(here + 8, here, 16, 32, 32)
    assert L.g5b_w4_dequantize(C.byref(x), 0, here, 32, None) == -1 and "multiple of 16" in _err()
    # host memory, or no device at all: never launched on
    x = _w4(here, here, 16, 32, 32)
    assert L.g5b_w4_dequantize(C.byref(x), 0, here, 32, None) == -1 and ("device" in _err())
    assert L.g5b_w4_matmul(None, here, 0, 1, 32, here, 16, here, 1 << 16, None) == -1 and "null" in _err()
    assert L.g5b_expert_sort(here, 1, 1, 1, here, here, here, None) == -1 and "device" in _err()


@pytest.mark.parametrize("T,topk,E", [(-1, 1, 1), (1, 0, 1), (1, 65, 1), (1, 1, 0), (1, 1, 1025), (1 << 20, 1, 1)])
def test_picks_out_of_range(T, topk, E):
    L, a = pkg.lib(), 1 << 20
    assert L.g5b_expert_sort(a, T, topk, E, a, a, a, None) == -1 and "outside" in _err()
    assert L.g5b_expert_gather(a, 0, T, 8, 8, a, a, topk, E, a, 8, None) == -1 and "outside" in _err()
    if E == 1:
        assert L.g5b_expert_combine(a, 0, 8, a, a, T, topk, 8, a, 8, None) == -1 and "outside" in _err()


def test_rows_out_of_range():
    L, a = pkg.lib(), 1 << 20
    assert L.g5b_expert_gather(a, 0, 1, 8, 7, a, a, 1, 1, a, 8, None) == -1 and "apart" in _err()
    assert L.g5b_expert_gather(a, 0, 1, 8, 8, a, a, 1, 1, a, 7, None) == -1 and "apart" in _err()
    assert L.g5b_expert_gather(a, 2, 1, 8, 8, a, a, 1, 1, a, 8, None) == -1 and "dtype 2" in _err()
    assert L.g5b_expert_combine(a, 0, 8, a, a, 1, 1, 8, a, 7, None) == -1 and "apart" in _err()


def test_workspace_sizes():
    m = _w4(1 << 20, 1 << 20, 4096, 4096, 128)
    L = pkg.lib()
    small, large = L.g5b_w4_matmul_workspace(C.byref(m), 0, 1), L.g5b_w4_matmul_workspace(C.byref(m), 0, 2048)
    assert 0 < small < large
    assert L.g5b_w4_matmul_workspace(C.byref(m), 1, 2048) < large
    assert L.g5b_w4_matmul_workspace(None, 0, 1) == 0 and L.g5b_w4_matmul_workspace(C.byref(m), 0, -1) == 0
    assert L.g5b_w4_experts_workspace(C.byref(m), C.byref(m), 0, 1, 0) == 0
    assert 0 < L.g5b_w4_experts_workspace(C.byref(m), C.byref(m), 0, 1, 8) < L.g5b_w4_experts_workspace(C.byref(m), C.byref(m), 0, 64, 8)


def test_python_checks():
    """Shapes, types and layouts that do not belong together end before the library is called."""
    rows, cols, group = 8, 70, 32
    codes, scales = torch.zeros((rows, 48), dtype=torch.uint8), torch.zeros((rows, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pkg.W4(codes[:, :40], scales, rows, cols, group)
    with pytest.raises(TypeError):
        pkg.W4(codes.int(), scales, rows, cols, group)
    with pytest.raises(ValueError):
        pkg.W4(codes, scales, rows, cols, 48)
    w = pkg.W4(codes, scales, rows, cols, group)
    assert w.count == 1
    x, ws = torch.zeros((3, cols)), torch.zeros(16)
    for bad in (torch.zeros((3, cols + 1)), torch.zeros((4, cols)), torch.zeros(cols), torch.zeros((cols, 3)).t()):
        with pytest.raises(ValueError):
            pkg.w4_matmul(w, bad, torch.zeros((3, rows)), ws, stream=0)
    with pytest.raises(TypeError):
        pkg.w4_matmul(w, x.half(), torch.zeros((3, rows)).half(), ws, stream=0)
    with pytest.raises(ValueError):
        pkg.w4_matmul(w, x, torch.zeros((3, rows), dtype=torch.bfloat16), ws, stream=0)
    with pytest.raises(RuntimeError):                      # host tensors: refused by the library
        pkg.w4_matmul(w, x, torch.zeros((3, rows)), ws, stream=0)
    with pytest.raises(ValueError):
        pkg.w4_quantize(torch.zeros((rows, cols), dtype=torch.uint8), w, stream=0)
    with pytest.raises(TypeError):
        pkg.w4_quantize(torch.zeros((rows, cols), dtype=torch.int32), w, stream=0)
    idx = torch.zeros((4, 2), dtype=torch.int32)
    with pytest.raises(TypeError):
        pkg.expert_sort(idx.long(), 3, idx.flatten(), idx, torch.zeros(4, dtype=torch.int32), stream=0)
    with pytest.raises(ValueError):
        pkg.expert_sort(idx, 3, idx.flatten(), idx, torch.zeros(3, dtype=torch.int32), stream=0)
    with pytest.raises(ValueError):
        pkg.expert_gather(torch.zeros((4, 8)), idx.flatten(), torch.zeros(4, dtype=torch.int32), torch.zeros((8, 9)), stream=0)


def test_experts_refusals():
    """Matrices that do not belong together, limits that are none, workspaces that are too small: before anything is launched."""
    L, a = pkg.lib(), 1 << 20
    m = lambda rows, cols, group=32, count=4: C.byref(_w4(a, a, rows, cols, group, count))       # noqa: E731

    def call(gate, up, down, limit=10.0, topk=2, T=1, dtype=0, ld=64):
        return L.g5b_w4_experts(gate, up, down, a, dtype, T, ld, a, a, topk, limit, a, ld, a, 1 << 30, None)
    # (without a device the addresses are refused first: then only that they are refused can be seen)
    device = L.g5b_device_count() > 0
    for args, kw, word in (((m(32, 64), m(32, 64, 64), m(64, 32)), {}, "belong together"), ((m(32, 64), m(33, 64), m(64, 32)), {}, "belong together"),
                           ((m(32, 64), m(32, 64), m(64, 33)), {}, "belong together"), ((m(32, 64), m(32, 64, 32, 3), m(64, 32)), {}, "matrices"),
                           ((m(32, 64), m(32, 64), m(64, 32)), {"limit": 0.0}, "limit"), ((m(32, 64), m(32, 64), m(64, 32)), {"limit": float("nan")}, "limit"),
                           ((m(32, 64), m(32, 64), m(64, 32)), {"topk": 65}, "picks"), ((m(32, 64), m(32, 64), m(64, 32)), {"ld": 63}, "apart"),
                           ((m(32, 64), m(32, 64), m(64, 32)), {"dtype": 2}, "dtype")):
        assert call(*args, **kw) == -1
        assert not device or word in _err() or "device" in _err()


def test_experts_refusals_say_what_is_wrong():
    """Every rule of the routed experts by its own message, whether there is a device or not: nothing but the addresses is wrong besides, and they are
    looked at last."""
    L, a = pkg.lib(), 1 << 20
    m = lambda rows, cols, group=32, count=4: C.byref(_w4(a, a, rows, cols, group, count))       # noqa: E731
    good = dict(gate=(32, 64), up=(32, 64), down=(64, 32), limit=10.0, topk=2, T=1, dtype=0, ldx=64, ldo=64, ws=1 << 30)

    def call(**kw):
        k = {**good, **kw}
        return L.g5b_w4_experts(m(*k["gate"]), m(*k["up"]), m(*k["down"]), a, k["dtype"], k["T"], k["ldx"], a, a, k["topk"], k["limit"], a, k["ldo"], a, k["ws"], None)
    for kw, word in (({"up": (32, 64, 64)}, "belong together"), ({"up": (33, 64)}, "belong together"), ({"up": (32, 65)}, "belong together"),
                     ({"down": (64, 33)}, "belong together"), ({"down": (65, 32)}, "belong together"), ({"up": (32, 64, 32, 3)}, "up holds 3 matrices"),
                     ({"down": (64, 32, 32, 5)}, "down holds 5 matrices"), ({"limit": 0.0}, "limit"), ({"limit": -1.0}, "limit"), ({"limit": float("nan")}, "limit"),
                     ({"topk": 0}, "picks"), ({"topk": 65}, "picks"), ({"T": -1}, "outside"), ({"T": (1 << 19) + 1}, "outside"), ({"ldx": 63}, "apart"), ({"ldo": 63}, "apart"),
                     ({"dtype": 2}, "dtype 2"), ({"gate": (32, 64, 48)}, "32, 64 or 128"), ({"gate": (0, 64)}, "outside")):
        assert call(**kw) == -1 and word in _err(), (kw, _err())
    for T in (1, 20, 100):                                 # picks one by one, by two, by 64
        need = L.g5b_w4_experts_workspace(m(32, 64), m(64, 32), 0, T, 2)
        assert call(T=T, ws=need - 1) == -1 and f"has {need - 1} bytes, {need} are needed" in _err()
        assert call(T=T, ws=need) == -1 and "device" in _err()
    assert call() == -1 and "device" in _err()
    assert call(down=(64, 32, 128)) == -1 and "device" in _err()          # groups of another size in the down matrix are fine


def test_product_refusals_say_what_is_wrong():
    L, a = pkg.lib(), 1 << 20
    w = C.byref(_w4(a, a, 16, 64, 32))

    def call(dtype=0, T=1, ldx=64, ldy=16, ws=1 << 30):
        return L.g5b_w4_matmul(w, a, dtype, T, ldx, a, ldy, a, ws, None)
    for kw, word in (({"dtype": 2}, "dtype 2"), ({"T": -1}, "outside"), ({"T": (1 << 19) + 1}, "outside"), ({"ldx": 63}, "apart"), ({"ldy": 15}, "apart")):
        assert call(**kw) == -1 and word in _err(), (kw, _err())
    for T in (1, 2, 5, 100):
        need = L.g5b_w4_matmul_workspace(w, 0, T)
        assert call(T=T, ws=need - 1) == -1 and f"has {need - 1} bytes, {need} are needed" in _err()
        assert call(T=T, ws=need) == -1 and "device" in _err()
    assert L.g5b_w4_dequantize(w, 0, a, 63, None) == -1 and "apart" in _err()
    assert L.g5b_w4_dequantize(w, 2, a, 64, None) == -1 and "dtype 2" in _err()
    src = lambda rows=16, cols=64, dtype=0, on=1: C.byref(pkg.Tensor(a, a, dtype, rows, cols, on))       # noqa: E731
    for t, blocks, word in ((src(on=0), (128, 128), "device tensor"), (src(rows=17), (128, 128), "17 x 64"), (src(cols=63), (128, 128), "16 x 63"),
                            (src(dtype=7), (128, 128), "dtype 7"), (src(dtype=pkg.DT_FP8), (0, 128), "scale blocks"), (src(dtype=pkg.DT_FP8), (128, -1), "scale blocks")):
        assert L.g5b_w4_quantize(t, *blocks, w, None) == -1 and word in _err(), _err()
    assert L.g5b_w4_quantize(src(), 128, 128, w, None) == -1 and "device" in _err()


def test_status_looks_on_the_current_stream(monkeypatch):
    """Where no stream is given: torch's current one of the current device, as for the calls whose waits it looks at."""
    asked = []
    monkeypatch.setattr(pkg, "_call_w4", lambda name, *args: asked.append((name, *args)))
    monkeypatch.setattr(pkg, "_raw_stream", lambda device: 1000 + device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    pkg.w4_status()
    pkg.w4_status(0)
    pkg.w4_status(stream=77)
    assert asked == [("g5b_w4_status", 1003), ("g5b_w4_status", 0), ("g5b_w4_status", 77)]
