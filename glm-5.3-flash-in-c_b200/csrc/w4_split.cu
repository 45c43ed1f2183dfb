// w4_split.cu - activation rows as F16 terms for the 4-bit products of many rows: x 2^e = hi + mid, exactly representable to 22 bits
// of the row's largest value (BF16 rows: hi alone, exact). Bound by memory: a row in, its terms out.
#include "w4.cuh"

namespace g5b {

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

}  // namespace g5b
