// w4_few.cu - 4-bit weights times a few activation rows: one decoded token, a small batch, the few tokens of an expert.
//
// Bound by HBM: half a byte and a scale's share per weight. The legacy matrix instruction does the products (16 weight rows x 16
// columns x 8 activation columns); the tensor memory's would need 128 rows at a time and hand-overs that cost more than the
// stream of a small matrix takes. A warp takes 16 rows; eight warps of a CTA share the row's blocks of 128 columns, so that all of a
// CTA's weights are asked for before the first is used, and their sums meet in shared memory in a fixed order.
//
//   codes   a lane loads 16 bytes of rows g and g + 8 (lane = 4 g + t), a quad 64 bytes: 128 columns of each. Nibbles become F16
//           pairs without a conversion: (code | 0x6400) is 1024 + code, (16 code | 0x6400) is 1024 + 16 code, and one packed operation
//           takes the offset (and the 16) off, exactly. A pair is columns i and i + 4 of a word's eight; which column stands for
//           which k of an MMA does not matter as long as both operands agree, and the activation terms lie in that order.
//   scales  in FP32, once per group, on the sums of the group. A quad's 128 columns are one group of 128; for smaller groups the
//           quad transposes its words first (two rounds of shuffles), so that every MMA pair is 32 columns of one group.
//   x       F32 rows are two F16 terms (22 significant bits of the row's largest), in columns of their own; BF16 rows one, exact.
// Sums are FP32: in the tensor cores over a group, outside across groups.
#include "common.cuh"
#include "mma_stage.cuh"
#include "w4.cuh"

namespace g5b {

// ------------------------------------------------------------------------- terms ----
__device__ __forceinline__ float x_value(const float *p) { return __ldg(p); }
__device__ __forceinline__ float x_value(const uint16_t *p) { return bf16_to_f32(__ldg(p)); }

// One CTA per row. The power of two brings the row's largest magnitude below 2^14; what falls below F16's 2^-24 then is 2^-38 of it.
template <typename IN, int TERMS>
__global__ void __launch_bounds__(256) w4_split_kernel(W4Terms t, const IN *x, size_t ldx, int cols, const int *n_rows, const int *order, int topk)
{
    __shared__ uint32_t s_max[8];
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.x;
    if (n_rows && row >= __ldg(n_rows)) return;
    const IN *xr = x + (size_t)(order ? __ldg(order + row) / topk : row) * ldx;
    uint32_t m = 0;
    for (int c = threadIdx.x; c < cols; c += 256) m = max(m, __float_as_uint(x_value(xr + c)) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, s_max[i]);
    const bool finite = m < 0x7f800000u;
    // 2^(e - 1) <= max < 2^e (a subnormal one counts as 2^-126)
    const int e = max((int)(m >> 23), 1) - 126, up = min(14 - e, 126);
    const float scale = __int_as_float((up + 127) << 23);
    if (threadIdx.x == 0) t.inv[row] = finite ? __int_as_float((127 - up) << 23) : __int_as_float(0x7fc00000);
    __half *hi = static_cast<__half *>(t.terms) + (size_t)row * TERMS * t.kp;
    for (int c0 = threadIdx.x * 8; c0 < t.kp; c0 += 256 * 8) {
        __align__(16) __half h[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = c0 + i, at = (i & 3) * 2 + (i >> 2);          // 0 4 1 5 2 6 3 7
            const float v = finite && c < cols ? x_value(xr + c) * scale : 0.f;
            h[at] = __float2half_rn(v);
            l[at] = __float2half_rn(v - __half2float(h[at]));
        }
        *reinterpret_cast<uint4 *>(hi + c0) = *reinterpret_cast<const uint4 *>(h);
        if (TERMS == 2) *reinterpret_cast<uint4 *>(hi + t.kp + c0) = *reinterpret_cast<const uint4 *>(l);
    }
}

void w4_split(cudaStream_t st, const W4Terms &t, const void *x, int dt, size_t ldx, int rows, int cols, const int *n_rows, const int *order, int topk,
              bool early)
{
    const float *f = static_cast<const float *>(x);
    const uint16_t *h = static_cast<const uint16_t *>(x);
#define SPLIT(IN, TERMS, p)                                                                                             \
    do {                                                                                                                \
        if (early) G5B_LAUNCH_PDL((w4_split_kernel<IN, TERMS>), dim3(rows), dim3(256), 0, st, t, p, ldx, cols, n_rows, order, topk); \
        else       G5B_LAUNCH((w4_split_kernel<IN, TERMS>), rows, 256, 0, st, t, p, ldx, cols, n_rows, order, topk);                 \
    } while (0)
    if (dt == DT_BF16) SPLIT(uint16_t, 1, h);
    else if (t.n_terms == 1) SPLIT(float, 1, f);
    else SPLIT(float, 2, f);
#undef SPLIT
}

// ---------------------------------------------------------------------- products ----
struct FewArgs {
    W4Mat w, up;
    const __half *terms;
    const float *inv;
    int kp, T, topk;
    const int *order;
    W4Slots slots;
    void *y;
    size_t ldy;
    int y_dt;
    float limit;
};

// the two F16 pairs (low nibbles, high nibbles) of a word's bytes 0 and 2, as code - 8
__device__ __forceinline__ void nibbles(uint32_t v, uint32_t &lo, uint32_t &hi)
{
    uint32_t a, b;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(a) : "r"(v));       // (v & mask) | 1024
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(b) : "r"(v));
    const __half2 l = __hadd2(*reinterpret_cast<__half2 *>(&a), __float2half2_rn(-1032.f));
    const __half2 h = __hfma2(*reinterpret_cast<__half2 *>(&b), __float2half2_rn(0.0625f), __float2half2_rn(-72.f));
    lo = *reinterpret_cast<const uint32_t *>(&l);
    hi = *reinterpret_cast<const uint32_t *>(&h);
}

// words of a quad: from "lane t holds words 0..3 of piece t" to "lane t holds word t of pieces 0..3"
__device__ __forceinline__ void quad_transpose(uint4 &v, int t)
{
    uint32_t x;
    const bool a = t & 1, b = t & 2;
    x = __shfl_xor_sync(0xffffffffu, a ? v.x : v.y, 1); if (a) v.x = x; else v.y = x;
    x = __shfl_xor_sync(0xffffffffu, a ? v.z : v.w, 1); if (a) v.z = x; else v.w = x;
    x = __shfl_xor_sync(0xffffffffu, b ? v.x : v.z, 2); if (b) v.x = x; else v.z = x;
    x = __shfl_xor_sync(0xffffffffu, b ? v.y : v.w, 2); if (b) v.y = x; else v.w = x;
}

__device__ __forceinline__ uint32_t word_of(const uint4 &v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

// WHOLE: groups of 128. NT: tiles of eight activation columns (terms of rows).
template <int TERMS, int NT, int MODE, bool WHOLE>
__global__ void __launch_bounds__(256) w4_few_kernel(const FewArgs a)
{
    constexpr int RT = MODE == W4_GATEUP ? 2 : 1, U = 4 / RT, ROWS = 8 * NT / TERMS, PITCH = 8 * NT + 1;
    __shared__ float s_sum[8][RT * 16][PITCH];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int r0 = blockIdx.x * 16;
    pdl_trigger();
    int first = blockIdx.y * ROWS, count = min(ROWS, a.T - first);
    size_t code_at = 0, scale_at = 0;
    if (MODE != W4_DENSE) {
        pdl_wait();                       // (the slots are another kernel's)
        if ((int)blockIdx.y >= __ldg(a.slots.n)) return;
        const int e = __ldg(a.slots.expert + blockIdx.y);
        first = __ldg(a.slots.first + blockIdx.y);
        count = __ldg(a.slots.count + blockIdx.y);
        code_at = (size_t)e * a.w.codes_stride;
        scale_at = (size_t)e * a.w.scales_stride;
    }
    const int blocks = a.kp / 128;
    const uint8_t *codes[RT][2];
    const uint16_t *scales[RT][2];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const W4Mat &w = i ? a.up : a.w;
            const int r = min(r0 + g + 8 * h, a.w.rows - 1);           // (a row behind the last: the last one's, not stored)
            codes[i][h] = w.codes + code_at + (size_t)r * w.pitch + 16 * t;
            scales[i][h] = w.scales + scale_at + (size_t)r * w.sp;
        }
    uint4 wv[U][RT][2];
    float sv[U][RT][2][WHOLE ? 1 : 4];
    auto load = [&](int b0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = b0 + 8 * u;
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    wv[u][i][h] = make_uint4(0u, 0u, 0u, 0u);
                    if (b * 64 + 16 * t < a.w.pitch) wv[u][i][h] = ld_stream16(codes[i][h] + b * 64);
                    if (WHOLE) sv[u][i][h][0] = b < blocks ? bf16_to_f32(__ldg(scales[i][h] + b)) : 0.f;
                    else {
                        // scales of the block's four pieces of 32 columns
                        const int per = a.w.group == 64 ? 1 : 0;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int k = (4 * b + j) >> per;
                            sv[u][i][h][WHOLE ? 0 : j] = k < a.w.groups ? bf16_to_f32(__ldg(scales[i][h] + k)) : 0.f;
                        }
                    }
                }
        }
    };
    load(warp);
    if (MODE == W4_DENSE) pdl_wait();
    const __half *bp[NT];
    bool live[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int col = n * 8 + g, i = col / TERMS;
        live[n] = i < count;
        const int at = !live[n] ? 0 : MODE == W4_GATEUP ? __ldg(a.order + first + i) / a.topk : first + i;
        bp[n] = a.terms + ((size_t)at * TERMS + col % TERMS) * a.kp + (WHOLE ? 32 : 8) * t;
    }
    float acc[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) acc[i][n][k] = 0.f;
    for (int b0 = warp; b0 < blocks; b0 += 8 * U) {
        if (b0 != warp) load(b0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = b0 + 8 * u;
            if (b >= blocks) break;
            if (!WHOLE) {
#pragma unroll
                for (int i = 0; i < RT; i++) { quad_transpose(wv[u][i][0], t); quad_transpose(wv[u][i][1], t); }
            }
            float c[RT][NT][4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint4 x[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    x[n] = make_uint4(0u, 0u, 0u, 0u);
                    if (live[n]) x[n] = *reinterpret_cast<const uint4 *>(bp[n] + b * 128 + (WHOLE ? 8 : 32) * j);
                }
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const uint32_t vg = word_of(wv[u][i][0], j), vh = word_of(wv[u][i][1], j);
                    uint32_t pg[4], ph[4];
                    nibbles(vg, pg[0], pg[1]); nibbles(vg >> 8, pg[2], pg[3]);
                    nibbles(vh, ph[0], ph[1]); nibbles(vh >> 8, ph[2], ph[3]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (j == 0 || !WHOLE) { c[i][n][0] = 0.f; c[i][n][1] = 0.f; c[i][n][2] = 0.f; c[i][n][3] = 0.f; }
                        mma_f16(c[i][n], pg[0], ph[0], pg[1], ph[1], x[n].x, x[n].y);
                        mma_f16(c[i][n], pg[2], ph[2], pg[3], ph[3], x[n].z, x[n].w);
                        if (j == 3 || !WHOLE) {
                            const float sg = sv[u][i][0][WHOLE ? 0 : j], sh = sv[u][i][1][WHOLE ? 0 : j];
                            acc[i][n][0] = fmaf(c[i][n][0], sg, acc[i][n][0]); acc[i][n][1] = fmaf(c[i][n][1], sg, acc[i][n][1]);
                            acc[i][n][2] = fmaf(c[i][n][2], sh, acc[i][n][2]); acc[i][n][3] = fmaf(c[i][n][3], sh, acc[i][n][3]);
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float *p = &s_sum[warp][i * 16 + g][n * 8 + 2 * t];
            p[0] = acc[i][n][0]; p[1] = acc[i][n][1];
            p[8 * PITCH] = acc[i][n][2]; p[8 * PITCH + 1] = acc[i][n][3];
        }
    __syncthreads();
    for (int o = threadIdx.x; o < 16 * count; o += 256) {
        const int r = o & 15, i = o >> 4;
        if (r0 + r >= a.w.rows) continue;
        float v[RT];
#pragma unroll
        for (int m = 0; m < RT; m++) {
            v[m] = 0.f;
#pragma unroll
            for (int w = 0; w < 8; w++)
#pragma unroll
                for (int k = TERMS - 1; k >= 0; k--) v[m] += s_sum[w][m * 16 + r][i * TERMS + k];
        }
        const int row = MODE == W4_GATEUP ? __ldg(a.order + first + i) / a.topk : first + i;
        const float inv = a.inv[row];
        float out = v[0] * inv;
        if (MODE == W4_GATEUP) out = swiglu_value(out, v[RT - 1] * inv, a.limit);
        const size_t at = (size_t)(first + i) * a.ldy + r0 + r;
        if (a.y_dt == DT_F32) static_cast<float *>(a.y)[at] = out;
        else static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(out);
    }
}

template <int TERMS, int NT, int MODE>
static int few_launch(cudaStream_t st, const W4Job &j)
{
    FewArgs a{j.w, j.up, static_cast<const __half *>(j.x.terms), j.x.inv, j.x.kp, j.T, j.topk, j.order, j.slots, j.y, j.ldy, j.y_dt, j.limit};
    constexpr int ROWS = 8 * NT / TERMS;
    const dim3 grid((j.w.rows + 15) / 16, j.mode == W4_DENSE ? (j.T + ROWS - 1) / ROWS : j.slots.max);
    if (j.w.group == 128) G5B_LAUNCH_PDL((w4_few_kernel<TERMS, NT, MODE, true>), grid, dim3(256), 0, st, a);
    else                  G5B_LAUNCH_PDL((w4_few_kernel<TERMS, NT, MODE, false>), grid, dim3(256), 0, st, a);
    return 0;
}
template <int TERMS, int NT>
static int few_mode(cudaStream_t st, const W4Job &j)
{
    return j.mode == W4_DENSE ? few_launch<TERMS, NT, W4_DENSE>(st, j) : j.mode == W4_GATEUP ? few_launch<TERMS, NT, W4_GATEUP>(st, j) : few_launch<TERMS, NT, W4_DOWN>(st, j);
}

// tiles of eight columns (terms of rows) for `rows` rows: 1, 2 or 4
static int few_tiles(int n_terms, int rows)
{
    const int n = (rows * n_terms + 7) / 8;
    return n <= 1 ? 1 : n <= 2 ? 2 : 4;
}
int w4_few_rows(int n_terms, int rows) { return 8 * few_tiles(n_terms, rows) / n_terms; }

int w4_few(cudaStream_t st, const W4Job &j)
{
    const int nt = few_tiles(j.x.n_terms, j.mode == W4_DENSE ? j.T : j.slots.rows);
    if (j.x.n_terms == 1) return nt == 1 ? few_mode<1, 1>(st, j) : nt == 2 ? few_mode<1, 2>(st, j) : few_mode<1, 4>(st, j);
    return nt == 1 ? few_mode<2, 1>(st, j) : nt == 2 ? few_mode<2, 2>(st, j) : few_mode<2, 4>(st, j);
}

}  // namespace g5b
