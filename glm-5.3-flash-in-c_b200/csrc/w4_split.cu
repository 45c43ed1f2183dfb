// w4_split.cu - activation rows as F16 terms for the 4-bit products of many rows: x 2^e = hi + mid, exactly representable to 22 bits
// of the row's largest value (BF16 rows: hi alone, exact). Bound by memory: a row in, its terms out.
#include <algorithm>

#include "w4.cuh"

namespace g5b {

// Rows one after the other by CTAs that fill the GPU once (a CTA for each of 16384 picks, of which 2048 were this rank's, took 30 us). The
// power of two brings a row's largest magnitude below 2^14; what falls below F16's 2^-24 then is 2^-38 of it.
template <typename IN, int TERMS>
__global__ void __launch_bounds__(256) w4_split_kernel(W4Terms t, const IN *x, size_t ldx, int rows, int cols, const int *n_rows, const int *order, int topk, bool wide)
{
    __shared__ uint32_t s_max[2][8];
    pdl_trigger();
    pdl_wait();
    if (n_rows) rows = min(rows, load_new(n_rows));
    int turn = 0;
    for (int row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
        const IN *xr = x + (size_t)(order ? load_new(order + row) / topk : row) * ldx;
        // the first 4096 columns stay in registers
        float first[2][8];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            w4_load8(first[i], xr, threadIdx.x * 8 + i * 2048, cols, wide);
#pragma unroll
            for (int k = 0; k < 8; k++) m = max(m, __float_as_uint(first[i][k]) & 0x7fffffffu);
        }
        for (int c = threadIdx.x * 8 + 4096; c < cols; c += 2048) {
            float v[8];
            w4_load8(v, xr, c, cols, wide);
#pragma unroll
            for (int k = 0; k < 8; k++) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
        }
        m = __reduce_max_sync(0xffffffffu, m);
        if ((threadIdx.x & 31) == 0) s_max[turn][threadIdx.x >> 5] = m;
        __syncthreads();                                          // (a row's maxima are not overwritten before everyone has read the next one's)
#pragma unroll
        for (int i = 0; i < 8; i++) m = max(m, s_max[turn][i]);
        const bool finite = m < 0x7f800000u;
        // 2^(e - 1) <= max < 2^e (a subnormal one counts as 2^-126)
        const int e = max((int)(m >> 23), 1) - 126, up = min(14 - e, 126);
        const float scale = __int_as_float((up + 127) << 23);
        if (threadIdx.x == 0) t.inv[row] = finite ? __int_as_float((127 - up) << 23) : __int_as_float(0x7fc00000);
        __half *hi = static_cast<__half *>(t.terms) + (size_t)row * TERMS * t.kp;
        auto put = [&](const float (&v)[8], int c) {
            __align__(16) __half h[8], l[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int to = (k & 3) * 2 + (k >> 2);            // 0 4 1 5 2 6 3 7
                const float f = finite ? v[k] * scale : 0.f;
                h[to] = __float2half_rn(f);
                l[to] = __float2half_rn(f - __half2float(h[to]));
            }
            *reinterpret_cast<uint4 *>(hi + c) = *reinterpret_cast<const uint4 *>(h);
            if (TERMS == 2) *reinterpret_cast<uint4 *>(hi + t.kp + c) = *reinterpret_cast<const uint4 *>(l);
        };
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (threadIdx.x * 8 + i * 2048 < t.kp) put(first[i], threadIdx.x * 8 + i * 2048);
        for (int c = threadIdx.x * 8 + 4096; c < t.kp; c += 2048) {
            float v[8];
            w4_load8(v, xr, c, cols, wide);
            put(v, c);
        }
    }
}

void w4_split(cudaStream_t st, const W4Terms &t, const void *x, int dt, size_t ldx, int rows, int cols, const int *n_rows, const int *order, int topk,
              bool early)
{
    const float *f = static_cast<const float *>(x);
    const uint16_t *h = static_cast<const uint16_t *>(x);
    const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * (dt == DT_F32 ? 4 : 2) % 16 == 0;
    const int grid = std::min(rows, 8 * dev_sms());
#define SPLIT(IN, TERMS, p)                                                                                             \
    do {                                                                                                                \
        if (early) G5B_LAUNCH_PDL((w4_split_kernel<IN, TERMS>), dim3(grid), dim3(256), 0, st, t, p, ldx, rows, cols, n_rows, order, topk, wide); \
        else       G5B_LAUNCH((w4_split_kernel<IN, TERMS>), grid, 256, 0, st, t, p, ldx, rows, cols, n_rows, order, topk, wide);                 \
    } while (0)
    if (dt == DT_BF16) SPLIT(uint16_t, 1, h);
    else SPLIT(float, 2, f);
#undef SPLIT
}

}  // namespace g5b
