// w4_ops.cu - the entry points of the 4-bit operators (include/glm53f_b200.h): checks of the arguments, workspaces, and
// the order of the launches.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <cuda.h>

#include "common.cuh"
#include "w4.h"

namespace g5b {
namespace {

constexpr int W4_MAX_ROWS = 1 << 22, W4_MAX_COLS = 1 << 17, W4_MAX_TOKENS = 1 << 19;
constexpr size_t WS_ALIGN = 256;

int fail(const char *fmt, ...)
{
    char msg[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof msg, fmt, ap);
    va_end(ap);
    set_last_error(msg);
    return -1;
}
int launched(const char *op)
{
    const cudaError_t rc = cudaGetLastError();
    return rc == cudaSuccess ? 0 : fail("%s: launch failed: %s", op, cudaGetErrorString(rc));
}

// Whether p is memory of the device `dev`: 1 yes, 0 no (`at`: which device's it is, -1 for the host's), -1 unknown. Asked of the
// driver: 0.04 us less an address than the runtime's call, and a product asks about five.
typedef CUresult (*PointerAttributesFn)(unsigned, CUpointer_attribute *, void **, CUdeviceptr);
int on_device(const void *p, int dev, int &at)
{
    static const PointerAttributesFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) { cudaGetLastError(); f = nullptr; }
        return reinterpret_cast<PointerAttributesFn>(f);
    }();
    unsigned type = 0, managed = 0;
    int ordinal = -1;
    CUpointer_attribute what[3] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL, CU_POINTER_ATTRIBUTE_IS_MANAGED};
    void *to[3] = {&type, &ordinal, &managed};
    at = -1;
    if (fn && fn(3, what, to, reinterpret_cast<CUdeviceptr>(p)) == CUDA_SUCCESS) {
        if (managed) return 1;
        if (type != CU_MEMORYTYPE_DEVICE) return 0;
        at = ordinal;
        return ordinal == dev;
    }
    cudaPointerAttributes a;                             // (a thread without a context, for instance)
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) { cudaGetLastError(); return -1; }
    if (a.type == cudaMemoryTypeManaged) return 1;
    if (a.type != cudaMemoryTypeDevice) return 0;
    at = a.device;
    return a.device == dev;
}
// Memory of the current device (where the launches go); `align`: what the kernels need of the address.
int check_ptr(const char *op, const char *what, const void *p, size_t align)
{
    if (!p) return fail("%s: %s is null", op, what);
    if (reinterpret_cast<uintptr_t>(p) % align) return fail("%s: %s must lie on a multiple of %zu bytes", op, what, align);
    int dev = -1, at = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); return fail("%s: no usable current CUDA device", op); }
    const int here = on_device(p, dev, at);
    if (here == 1) return 0;
    if (here < 0) return fail("%s: no usable current CUDA device", op);
    return at < 0 ? fail("%s: %s is not device memory", op, what) : fail("%s: %s lies on device %d, the current one is %d", op, what, at, dev);
}
int elt(int dt) { return dt == DT_F32 ? 4 : 2; }
int check_dtype(const char *op, int dt) { return dt == DT_F32 || dt == DT_BF16 ? 0 : fail("%s: rows are F32 or BF16, not dtype %d", op, dt); }

// Every entry point looks at sizes, types and distances first, then at the workspace's size, and at addresses last.
int check_mat(const char *op, const char *what, const g5b_w4 *m, int count, W4Mat &w)
{
    if (!m) return fail("%s: %s is null", op, what);
    if (m->rows < 1 || m->rows > W4_MAX_ROWS || m->cols < 1 || m->cols > W4_MAX_COLS)
        return fail("%s: %s of %d x %d is outside 1 x 1 .. %d x %d", op, what, m->rows, m->cols, W4_MAX_ROWS, W4_MAX_COLS);
    if (m->group != 32 && m->group != 64 && m->group != 128) return fail("%s: groups of %s have 32, 64 or 128 columns, not %d", op, what, m->group);
    if (m->count < 1 || m->count > G5B_MAX_EXPERTS || (count && m->count != count)) return fail("%s: %s holds %d matrices", op, what, m->count);
    w.codes = m->codes; w.scales = m->scales;
    w.rows = m->rows; w.cols = m->cols; w.group = m->group;
    w.pitch = (int)g5b_w4_pitch(m->cols); w.sp = (int)g5b_w4_scale_pitch(m->cols, m->group);
    w.groups = (m->cols + m->group - 1) / m->group;
    w.codes_stride = (size_t)w.rows * w.pitch; w.scales_stride = (size_t)w.rows * w.sp;
    return 0;
}
int check_mat_ptr(const char *op, const char *what, const W4Mat &w)
{
    return check_ptr(op, what, w.codes, 16) || check_ptr(op, what, w.scales, 16) ? -1 : 0;
}

// Pieces of a workspace, one after the other; without memory behind it a count of the bytes.
struct Pieces {
    uint8_t *base;
    size_t used = 0;
    template <typename T> T *take(size_t n)
    {
        T *p = base ? reinterpret_cast<T *>(base + used) : nullptr;
        used += (n * sizeof(T) + WS_ALIGN - 1) / WS_ALIGN * WS_ALIGN;
        return p;
    }
};
W4Terms terms_of(Pieces &ws, int n_terms, int cols, size_t rows)
{
    W4Terms t;
    t.n_terms = n_terms; t.kp = w4_kp(cols);
    t.terms = ws.take<uint16_t>(rows * n_terms * t.kp);
    t.inv = ws.take<float>(rows);
    return t;
}
int check_ws(const char *op, size_t have, size_t need)
{
    return have >= need ? 0 : fail("%s: the workspace has %zu bytes, %zu are needed", op, have, need);
}

// How a call of the experts goes: PICKS (every pick on its own, nothing is sorted), FEW (w4_few on sorted picks), MANY (w4_many) or EITHER.
// PICKS saves the sort, 7 us, and reads an expert twice that two picks have, 2 us each: n picks of E experts have n^2 / 2E such pairs
// (three tokens of 288 experts 70.2 -> 63.6 us, four 84.5 -> 77.2).
// FEW reads an expert's weights for every two rows, MANY once, at the speed of its conversion: 1 row to an expert 604 against 835 us,
// 2 818 against 968, 2.8 the same (F32).
// How many picks are here only the device knows: of a rank's call one in eight may be. EITHER: the sort chooses, and the other kind's
// kernels find nothing to do, 4 us in all (a rank of 36 experts: 32 tokens 135 us by w4_many, 101 so; 64 tokens 160 and 139, BF16 145 and 141).
enum { PICKS, FEW, MANY, EITHER };
struct ExpertsPlan { int how, rows; };           // rows of a slot at most
constexpr int PICKS_ALWAYS = 16, PICKS_MOST = 32, RANKS = 8;
ExpertsPlan experts_plan(int T, int topk, int E, int H, int I)
{
    const int n = T * topk, h = w4_few_rows(H), i = w4_few_rows(I), rows = h < i ? h : i;
    if (rows && n <= PICKS_MOST && (n <= PICKS_ALWAYS || n * n <= 4 * E)) return {PICKS, 1};
    if (rows > 1 && n <= rows * E) return {FEW, rows};
    if (rows > 1 && n <= RANKS * rows * E) return {EITHER, rows};
    return {MANY, W4_MANY_ROWS};
}
struct ExpertsWs {
    int *order, *place, *offsets;
    W4Slots slots;
    W4Terms x, h;
    float *act, *rows;
};
ExpertsWs experts_ws(Pieces &ws, const ExpertsPlan &plan, int n_terms, int T, int topk, int E, int H, int I)
{
    ExpertsWs w{};
    const size_t n = (size_t)T * topk;
    if (plan.how != PICKS) {
        w.order = ws.take<int>(n); w.place = ws.take<int>(n); w.offsets = ws.take<int>(E + 1);
        w.slots.rows = plan.rows;
        if (plan.how == EITHER) { w.slots.many_rows = W4_MANY_ROWS; w.slots.few_most = plan.rows * E; }
        w.slots.max = (int)(n / plan.rows + (n < (size_t)E ? n : (size_t)E));
        w.slots.n = ws.take<int>(3);
        w.slots.expert = ws.take<int>(w.slots.max); w.slots.first = ws.take<int>(w.slots.max); w.slots.count = ws.take<int>(w.slots.max);
    }
    if (plan.how == MANY || plan.how == EITHER) {
        w.x = terms_of(ws, n_terms, H, n);
        w.h = terms_of(ws, 2, I, n);                // (FP32 rows, whatever the caller's are)
    }
    w.act = ws.take<float>(n * I);
    w.rows = ws.take<float>(n * H);
    return w;
}

}  // namespace
}  // namespace g5b

using namespace g5b;

extern "C" size_t g5b_w4_pitch(int cols) { return cols < 1 ? 0 : (size_t)(cols + 31) / 32 * 16; }
extern "C" size_t g5b_w4_scale_pitch(int cols, int group)
{
    if (cols < 1 || (group != 32 && group != 64 && group != 128)) return 0;
    return (size_t)((cols + group - 1) / group + 7) / 8 * 8;
}

extern "C" int g5b_w4_quantize(const g5b_tensor *src, int br, int bc, const g5b_w4 *dst, void *stream)
{
    const char *op = "g5b_w4_quantize";
    W4Mat w;
    if (check_mat(op, "the matrix", dst, 1, w)) return -1;
    if (!src || !src->on_device) return fail("%s: the source must be a device tensor", op);
    if (src->rows != w.rows || src->cols != w.cols) return fail("%s: a source of %d x %d for a matrix of %d x %d", op, src->rows, src->cols, w.rows, w.cols);
    if (src->dtype != DT_F32 && src->dtype != DT_BF16 && src->dtype != DT_FP8) return fail("%s: dtype %d of the source", op, src->dtype);
    if (src->dtype == DT_FP8 && (br < 1 || bc < 1)) return fail("%s: scale blocks of %d x %d", op, br, bc);
    if (check_mat_ptr(op, "the matrix", w) || check_ptr(op, "the source", src->data, src->dtype == DT_F32 ? 4 : src->dtype == DT_BF16 ? 2 : 1)) return -1;
    if (src->dtype == DT_FP8 && check_ptr(op, "the scale grid", src->scale_inv, 4)) return -1;
    w4_quantize(static_cast<cudaStream_t>(stream), w, src->data, src->dtype, src->scale_inv, br, bc);
    return launched(op);
}

extern "C" int g5b_w4_dequantize(const g5b_w4 *m, int dtype, void *out, size_t ldo, void *stream)
{
    const char *op = "g5b_w4_dequantize";
    W4Mat w;
    if (check_mat(op, "the matrix", m, 1, w) || check_dtype(op, dtype)) return -1;
    if (ldo < (size_t)w.cols) return fail("%s: rows %zu apart for %d columns", op, ldo, w.cols);
    if (check_mat_ptr(op, "the matrix", w) || check_ptr(op, "the output", out, elt(dtype))) return -1;
    w4_dequantize(static_cast<cudaStream_t>(stream), w, out, dtype, ldo);
    return launched(op);
}

extern "C" size_t g5b_w4_matmul_workspace(const g5b_w4 *m, int dtype, int T)
{
    if (!m || m->cols < 1 || m->cols > W4_MAX_COLS || T < 0 || T > W4_MAX_TOKENS) return 0;
    Pieces ws{nullptr};
    const int n_terms = dtype == DT_BF16 ? 1 : 2;
    if (w4_few_takes(m->cols, T)) return WS_ALIGN;
    terms_of(ws, n_terms, m->cols, T);
    ws.take<float>(w4_many_part_floats(m->rows, m->cols, T));
    return ws.used;
}

extern "C" int g5b_w4_matmul(const g5b_w4 *m, const void *x, int dtype, int T, size_t ldx, void *y, size_t ldy, void *workspace,
                             size_t workspace_bytes, void *stream)
{
    const char *op = "g5b_w4_matmul";
    W4Job j{};
    if (check_mat(op, "the matrix", m, 1, j.w) || check_dtype(op, dtype)) return -1;
    if (T < 0 || T > W4_MAX_TOKENS) return fail("%s: %d rows are outside 0 .. %d", op, T, W4_MAX_TOKENS);
    if (T && (ldx < (size_t)j.w.cols || ldy < (size_t)j.w.rows)) return fail("%s: rows %zu and %zu apart for a matrix of %d x %d", op, ldx, ldy, j.w.rows, j.w.cols);
    if (T && check_ws(op, workspace_bytes, g5b_w4_matmul_workspace(m, dtype, T))) return -1;
    if (check_mat_ptr(op, "the matrix", j.w)) return -1;
    if (T == 0) return 0;
    if (check_ptr(op, "x", x, elt(dtype)) || check_ptr(op, "y", y, elt(dtype)) || check_ptr(op, "the workspace", workspace, WS_ALIGN)) return -1;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Pieces ws{static_cast<uint8_t *>(workspace)};
    j.mode = W4_DENSE; j.T = T; j.count = 1;
    j.y = y; j.ldy = ldy; j.y_dt = dtype;
    if (w4_few_takes(j.w.cols, T)) {
        j.x = x; j.x_dt = dtype; j.ldx = ldx;
        return w4_few(st, j) ? -1 : launched(op);
    }
    j.terms = terms_of(ws, dtype == DT_BF16 ? 1 : 2, j.w.cols, T);
    w4_split(st, j.terms, x, dtype, ldx, T, j.w.cols, nullptr, nullptr, 1, false);
    return w4_many(st, j, ws.take<float>(w4_many_part_floats(j.w.rows, j.w.cols, T))) ? -1 : launched(op);
}

static int check_picks(const char *op, int T, int topk, int n_experts)
{
    if (T < 0 || T > W4_MAX_TOKENS || topk < 1 || topk > G5B_MAX_TOPK) return fail("%s: %d tokens with %d picks are outside 0 .. %d with 1 .. %d", op, T, topk, W4_MAX_TOKENS, G5B_MAX_TOPK);
    if (n_experts < 1 || n_experts > G5B_MAX_EXPERTS) return fail("%s: %d experts are outside 1 .. %d", op, n_experts, G5B_MAX_EXPERTS);
    return 0;
}

extern "C" int g5b_expert_sort(const int32_t *idx, int T, int topk, int n_experts, int32_t *order, int32_t *place, int32_t *offsets, void *stream)
{
    const char *op = "g5b_expert_sort";
    if (check_picks(op, T, topk, n_experts) || check_ptr(op, "offsets", offsets, 4)) return -1;
    if (T == 0) return cudaMemsetAsync(offsets, 0, (size_t)(n_experts + 1) * 4, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : launched(op);
    if (check_ptr(op, "idx", idx, 4) || check_ptr(op, "order", order, 4) || check_ptr(op, "place", place, 4)) return -1;
    if (expert_sort(static_cast<cudaStream_t>(stream), idx, T, topk, n_experts, order, place, offsets, nullptr)) return launched(op), -1;
    return launched(op);
}

extern "C" int g5b_expert_gather(const void *x, int dtype, int T, int cols, size_t ldx, const int32_t *order, const int32_t *offsets, int topk,
                                 int n_experts, void *rows, size_t ldr, void *stream)
{
    const char *op = "g5b_expert_gather";
    if (check_picks(op, T, topk, n_experts) || check_dtype(op, dtype)) return -1;
    if (cols < 1 || cols > W4_MAX_COLS || ldx < (size_t)cols || ldr < (size_t)cols) return fail("%s: rows %zu and %zu apart for %d columns", op, ldx, ldr, cols);
    if (T == 0) return 0;
    if (check_ptr(op, "x", x, elt(dtype)) || check_ptr(op, "order", order, 4) || check_ptr(op, "offsets", offsets, 4) || check_ptr(op, "rows", rows, elt(dtype))) return -1;
    const size_t b = elt(dtype);
    expert_gather(static_cast<cudaStream_t>(stream), x, cols * b, ldx * b, ldr * b, order, offsets, T * topk, topk, n_experts, rows);
    return launched(op);
}

extern "C" int g5b_expert_combine(const void *rows, int dtype, size_t ldr, const int32_t *place, const float *weights, int T, int topk, int cols,
                                  void *out, size_t ldo, void *stream)
{
    const char *op = "g5b_expert_combine";
    if (check_picks(op, T, topk, 1) || check_dtype(op, dtype)) return -1;
    if (cols < 1 || cols > W4_MAX_COLS || ldr < (size_t)cols || ldo < (size_t)cols) return fail("%s: rows %zu and %zu apart for %d columns", op, ldr, ldo, cols);
    if (T == 0) return 0;
    if (check_ptr(op, "rows", rows, elt(dtype)) || check_ptr(op, "place", place, 4) || check_ptr(op, "out", out, elt(dtype))) return -1;
    if (weights && check_ptr(op, "weights", weights, 4)) return -1;
    expert_combine(static_cast<cudaStream_t>(stream), rows, dtype, ldr, place, 0, weights, T, topk, cols, out, dtype, ldo, false);
    return launched(op);
}

extern "C" size_t g5b_w4_experts_workspace(const g5b_w4 *gate, const g5b_w4 *down, int dtype, int T, int topk)
{
    if (!gate || !down || T < 0 || T > W4_MAX_TOKENS || topk < 1 || topk > G5B_MAX_TOPK || gate->count < 1 || gate->count > G5B_MAX_EXPERTS ||
        gate->cols < 1 || gate->cols > W4_MAX_COLS || down->cols < 1 || down->cols > W4_MAX_COLS)
        return 0;
    Pieces ws{nullptr};
    const int n_terms = dtype == DT_BF16 ? 1 : 2, rows = T < 1 ? 1 : T;
    experts_ws(ws, experts_plan(rows, topk, gate->count, gate->cols, down->cols), n_terms, rows, topk, gate->count, gate->cols, down->cols);
    return ws.used;
}

extern "C" int g5b_w4_experts(const g5b_w4 *gate, const g5b_w4 *up, const g5b_w4 *down, const void *x, int dtype, int T, size_t ldx,
                              const int32_t *idx, const float *weights, int topk, float limit, void *out, size_t ldo, void *workspace,
                              size_t workspace_bytes, void *stream)
{
    const char *op = "g5b_w4_experts";
    W4Mat wg, wu, wd;
    if (check_mat(op, "gate", gate, 0, wg) || check_mat(op, "up", up, gate->count, wu) || check_mat(op, "down", down, gate->count, wd)) return -1;
    if (wu.rows != wg.rows || wu.cols != wg.cols || wu.group != wg.group || wd.rows != wg.cols || wd.cols != wg.rows)
        return fail("%s: gate %d x %d, up %d x %d and down %d x %d do not belong together", op, wg.rows, wg.cols, wu.rows, wu.cols, wd.rows, wd.cols);
    if (check_picks(op, T, topk, gate->count) || check_dtype(op, dtype)) return -1;
    if (!(limit > 0.f)) return fail("%s: the clamp's limit must be above zero (infinity for none)", op);
    if (ldx < (size_t)wg.cols || ldo < (size_t)wg.cols) return fail("%s: rows %zu and %zu apart for %d columns", op, ldx, ldo, wg.cols);
    if (T && check_ws(op, workspace_bytes, g5b_w4_experts_workspace(gate, down, dtype, T, topk))) return -1;
    if (check_mat_ptr(op, "gate", wg) || check_mat_ptr(op, "up", wu) || check_mat_ptr(op, "down", wd)) return -1;
    if (T == 0) return 0;
    if (check_ptr(op, "x", x, elt(dtype)) || check_ptr(op, "idx", idx, 4) || check_ptr(op, "weights", weights, 4) || check_ptr(op, "out", out, elt(dtype)) ||
        check_ptr(op, "the workspace", workspace, WS_ALIGN))
        return -1;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int E = gate->count, H = wg.cols, I = wg.rows, n = T * topk, n_terms = dtype == DT_BF16 ? 1 : 2;
    Pieces pieces{static_cast<uint8_t *>(workspace)};
    const ExpertsPlan plan = experts_plan(T, topk, E, H, I);
    const ExpertsWs ws = experts_ws(pieces, plan, n_terms, T, topk, E, H, I);
    W4Job j{};
    j.count = E; j.T = n; j.order = ws.order; j.topk = topk; j.slots = ws.slots; j.limit = limit; j.y_dt = DT_F32;
    if (plan.how != PICKS && expert_sort(st, idx, T, topk, E, ws.order, ws.place, ws.offsets, &ws.slots)) return launched(op), -1;
    const bool few = plan.how != MANY, many = plan.how == MANY || plan.how == EITHER;
    W4Slots many_slots = ws.slots;
    const int *many_n = ws.offsets + E;                        // picks that the products of many rows take
    if (plan.how == EITHER) { many_slots.n = ws.slots.n + 1; many_slots.rows = W4_MANY_ROWS; many_n = ws.slots.n + 2; }
    if (many) w4_split(st, ws.x, x, dtype, ldx, n, H, many_n, ws.order, topk, false);
    // The first of the kernels that may start early (their weights, which no kernel before them in this call writes) comes behind one that
    // was launched the ordinary way: whatever the stream held before the call is over by then.
    j.mode = W4_GATEUP; j.w = wg; j.up = wu; j.y = ws.act; j.ldy = I;
    j.x = x; j.x_dt = dtype; j.ldx = ldx; j.terms = ws.x;
    j.idx = plan.how == PICKS ? idx : nullptr; j.early = plan.how != PICKS;
    W4Job jm = j;
    jm.slots = many_slots;
    if ((few && w4_few(st, j)) || (many && w4_many(st, jm, nullptr))) return -1;
    if (many) w4_split(st, ws.h, ws.act, DT_F32, I, n, I, many_n, nullptr, 1, true);
    j.mode = W4_DOWN; j.w = wd; j.y = ws.rows; j.ldy = H;
    j.x = ws.act; j.x_dt = DT_F32; j.ldx = I; j.terms = ws.h; j.early = true;
    jm = j;
    jm.slots = many_slots;
    if ((few && w4_few(st, j)) || (many && w4_many(st, jm, nullptr))) return -1;
    expert_combine(st, ws.rows, DT_F32, H, plan.how == PICKS ? idx : ws.place, plan.how == PICKS ? E : 0, weights, T, topk, H, out, dtype, ldo, true);
    return launched(op);
}

extern "C" int g5b_w4_status(void *stream)
{
    const int few = w4_few_status(static_cast<cudaStream_t>(stream)), many = w4_many_status(static_cast<cudaStream_t>(stream)), code = few ? few : many;
    if (few < 0 || many < 0) return launched("g5b_w4_status"), -1;
    return code ? fail("g5b_w4_status: a wait of a 4-bit product ran out (code %d): results since the last look are undefined", code) : 0;
}
