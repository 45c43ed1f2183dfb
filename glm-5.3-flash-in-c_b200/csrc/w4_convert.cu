// w4_convert.cu - a matrix to 4-bit codes with group scales, and its values back.
//
// Per row and group m = max |w|, s = bf16(m / 7), code = 8 + clamp(round(w / s), -7, 7), halves to even, both roundings of s to
// nearest even. The quotient is taken exactly. A BF16 weight's (both have 8 significant bits) is a half or at least 2^-10 away from one, so
// the product with 1 / s, 2^-21 off at most, is first rounded to a multiple of 2^-11 and then to an integer. Of FP32 values the product
// decides, and where it lies near a half the residual w - q s does, which is exact there (q s has 12 significant bits; within half a step
// of it the difference loses none). A division instead is twenty instructions a weight, as many as the SM can issue while HBM delivers
// an FP8 weight.
//
// Both directions are bound by HBM, the first nearly by the instructions a weight takes. There a lane takes 32 columns, so that what
// is paid per group - the division, the reciprocal, the maximum's shuffles - is paid once for 32 weights, and its codes are one store;
// eight columns a lane paid it four times, converted to integers by the slow instruction, and took 72 us for 12288 x 4096 BF16 weights. (With
// residuals for BF16 weights too, every second warp met an exact half: 42 us.) Both directions of those together take 55.8 us, 6.3 TB/s.
#include "w4.cuh"

namespace g5b {

constexpr int CV_WARPS = 8;
constexpr int CV_COLS = 1024;      // columns a warp takes

// Eight values from column c0 on, of rows that allow 16-byte loads (8 of FP8): zero behind the last column, which no load crosses.
template <int DT>
__device__ __forceinline__ void load8(float (&v)[8], const void *src, size_t at, int c0, int cols)
{
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.f;
    if (c0 >= cols) return;
    if (DT == DT_F32) {
        const float4 a = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(src) + at));
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        if (c0 + 4 >= cols) return;
        const float4 b = __ldcs(reinterpret_cast<const float4 *>(static_cast<const float *>(src) + at + 4));
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else if (DT == DT_BF16) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(src) + at));
        bf16x2_to_f32(a.x, v[0], v[1]); bf16x2_to_f32(a.y, v[2], v[3]); bf16x2_to_f32(a.z, v[4], v[5]); bf16x2_to_f32(a.w, v[6], v[7]);
    } else {
        const uint2 a = __ldcs(reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(src) + at));
        e4m3x4_to_f32(a.x, v[0], v[1], v[2], v[3]);
        e4m3x4_to_f32(a.y, v[4], v[5], v[6], v[7]);
    }
}
// A lane's 32 values of rows that lie anyhow: the warp brings its n elements from e0 on into shared memory in words, as they lie in memory, and a lane
// shifts its own out of them, from element `start` of those on, S words and a part of one more; zero behind the first `valid`. A word of padding to S keeps lanes in different banks. (An element at a time, the lanes 32
// columns apart: 6319 x 2649 BF16 weights there and back 80 us.)
template <int DT> constexpr int cv_words = DT == DT_F32 ? 32 : DT == DT_BF16 ? 16 : 8;
template <int DT> constexpr int cv_room = 33 * (cv_words<DT> + 1);
template <int DT>
__device__ __forceinline__ void load32(float (&v)[4][8], const uint8_t *src, size_t bytes, size_t e0, int n, int start, int valid, uint32_t *room)
{
    constexpr int SIZE = DT == DT_F32 ? 4 : DT == DT_BF16 ? 2 : 1, S = cv_words<DT>, LOG = DT == DT_F32 ? 5 : DT == DT_BF16 ? 4 : 3;
    const int lane = threadIdx.x & 31;
    const uint8_t *first = src + e0 * SIZE;
    const int off = (int)(reinterpret_cast<uintptr_t>(first) & 3u), words = n > 0 ? (off + n * SIZE + 3) / 4 : 0;
    const uint8_t *base = first - off;
    // (where the matrix begins or ends within a word, that one's bytes singly)
    const int w0 = base < src, w1 = words - (words > 0 && base + 4 * (size_t)words > src + bytes);
#pragma unroll 8
    for (int w = w0 + lane; w < w1; w += 32) room[w + (w >> LOG)] = __ldcs(reinterpret_cast<const uint32_t *>(base) + w);
    if (lane < 2 && words > 0 && (lane ? w1 < words : w0 > 0)) {
        const int w = lane ? words - 1 : 0;
        uint32_t x = 0;
        for (int b = 0; b < 4; b++) {
            const uint8_t *at = base + 4 * (size_t)w + b;
            if (at >= src && at < src + bytes) x |= (uint32_t)*at << (8 * b);
        }
        room[w + (w >> LOG)] = x;
    }
    __syncwarp();
    const int at = off + start * SIZE, word = at >> 2;
    const uint32_t shift = 8u * (uint32_t)(at & 3);
    uint32_t a = room[word + (word >> LOG)];
    float *out = &v[0][0];
#pragma unroll
    for (int k = 0; k < S; k++) {
        const int next = word + k + 1;
        const uint32_t b = room[next + (next >> LOG)], u = __funnelshift_r(a, b, shift);
        if (DT == DT_F32) out[k] = __uint_as_float(u);
        else if (DT == DT_BF16) bf16x2_to_f32(u, out[2 * k], out[2 * k + 1]);
        else e4m3x4_to_f32(u, out[4 * k], out[4 * k + 1], out[4 * k + 2], out[4 * k + 3]);
        a = b;
    }
    if (valid < 32)
#pragma unroll
        for (int k = 0; k < 32; k++) if (k >= valid) out[k] = 0.f;
}

// (five CTAs to an SM: 12288 x 4096 FP8 weights there and back 73.8 -> 70.2 us; six spill)
template <int DT, bool WHOLE, bool NARROW>
__global__ void __launch_bounds__(CV_WARPS * 32, 5) w4_quantize_kernel(W4Mat w, uint8_t *codes, uint16_t *scales, const void *src, const float *inv,
                                                                    int br, int bc, int scols, unsigned pieces, int narrow_log)
{
    const int lane = threadIdx.x & 31;
    const unsigned unit = blockIdx.x * CV_WARPS + (threadIdx.x >> 5), row_ = unit / pieces;
    // Rows of up to 512 columns (NARROW) share a warp: 2^narrow_log lanes to one (16357 x 161 FP8 weights there and back in a warp each 35.0 us, so 18.7).
    const int lanes_log = NARROW ? narrow_log : 5;
    const int per_warp = 32 >> lanes_log, row0 = (int)row_ * per_warp, p0 = (int)(unit - row_ * pieces) * CV_COLS;
    if (row0 >= w.rows) return;
    const int own = lane >> lanes_log, c0 = p0 + (lane - (own << lanes_log)) * 32, per = w.group / 32;
    const bool exists = row0 + own < w.rows;
    const int row = exists ? row0 + own : w.rows - 1, cols = exists ? w.cols : 0;         // (a lane without a row takes zeros)
    float v[4][8];
    if constexpr (!WHOLE) {
        __shared__ uint32_t room[CV_WARPS][cv_room<DT>];
        constexpr int SIZE = DT == DT_F32 ? 4 : DT == DT_BF16 ? 2 : 1;
        const int n = per_warp == 1 ? min(CV_COLS, w.cols - p0) : min(per_warp, w.rows - row0) * w.cols;
        load32<DT>(v, static_cast<const uint8_t *>(src), (size_t)w.rows * w.cols * SIZE, (size_t)row0 * w.cols + p0, n, own * w.cols + c0 - p0, cols - c0,
                   room[threadIdx.x >> 5]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int c = c0 + 8 * i;
        if constexpr (WHOLE) load8<DT>(v[i], src, (size_t)row * w.cols + c, c, cols);
        if (DT == DT_FP8) {
            // the weight is the FP32 product of code and block scale
            const float *irow = inv + (size_t)(row / br) * scols;
            if (bc % 8 == 0) {
                const float s = c < cols ? __ldg(irow + c / bc) : 0.f;
#pragma unroll
                for (int k = 0; k < 8; k++) v[i][k] = __fmul_rn(v[i][k], s);
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) if (c + k < cols) v[i][k] = __fmul_rn(v[i][k], __ldg(irow + (c + k) / bc));
            }
        }
    }
    // the largest magnitude as bits: infinities and NaN are above every number
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int k = 0; k < 8; k++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(v[i][k])));
    uint32_t m = __float_as_uint(most);
    for (int o = 1; o < per; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool finite = m < 0x7f800000u;
    const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(__uint_as_float(m), 7.0f));
    const float s = __bfloat162float(sb);
    const bool live = finite && s > 0.f;
    // 1 / s of a small s may be infinite: the quotient is then taken of both times 2^64 (the long way)
    const bool tiny = s < 0x1p-100f;
    const float up = tiny ? 0x1p64f : 1.0f, su = s * up, r = live ? __frcp_rn(su) : 0.f, half = 0.5f * su;
    // Rounded by adding 1.5 2^23 + 8, in whose low bits the code then lies; eight codes are put together by multiplications, the same pipe. A
    // quotient over 7.5 (of a scale rounded to a few bits) and FP32 residuals from half a step on take the long way, eight weights at a time.
    constexpr float MAGIC = 12582912.0f + 8.0f;
    constexpr uint32_t MAGIC_BITS = 0x4b400000u, ONES = 0x11111111u;
    constexpr float STEP = 6144.0f;                          // 1.5 2^12, from where on FP32 numbers are 2^-11 apart
    const bool clamp = tiny || __uint_as_float(m) > 7.5f * s;
    __align__(16) uint32_t packed[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t word = 0u - MAGIC_BITS * ONES;
        float far = 0.f;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            float t;
            if (DT == DT_BF16) t = __fadd_rn(fmaf(v[i][k], r, STEP), MAGIC - STEP);
            else {
                t = fmaf(v[i][k], r, MAGIC);
                far = fmaxf(far, fabsf(fmaf(-(t - MAGIC), su, v[i][k])));
            }
            word += __float_as_uint(t) << (4 * k);
        }
        if (clamp || (DT != DT_BF16 && far >= half)) {
            word = 0u;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float x = v[i][k] * up, t = fmaf(x, r, MAGIC), q = t - MAGIC, d = fmaf(-q, su, x), ad = fabsf(d);
                int n = (int)(__float_as_uint(t) - MAGIC_BITS);                   // the code
                // one step on where the residual is over half a step, or half a step and the integer odd
                if (ad > half || (ad == half && (n & 1))) n += d > 0.f ? 1 : -1;
                word |= (uint32_t)min(max(n, 1), 15) << (4 * k);
            }
        }
        packed[i] = live ? word : 0x88888888u;
    }
    if (!exists) return;
    if (c0 / 2 < w.pitch) *reinterpret_cast<uint4 *>(codes + (size_t)row * w.pitch + c0 / 2) = *reinterpret_cast<const uint4 *>(packed);
    const int group = c0 / w.group;
    if ((lane & (per - 1)) == 0 && group < w.sp)
        scales[(size_t)row * w.sp + group] = group >= w.groups ? (uint16_t)0 : finite ? __bfloat16_as_ushort(sb) : (uint16_t)0x7fc0;
    if (per_warp > 1)                             // (scales behind what these lanes cover)
        for (int g = (1 << lanes_log) / per + (c0 >> 5); g < w.sp; g += 1 << lanes_log) scales[(size_t)row * w.sp + g] = 0;
}

void w4_quantize(cudaStream_t st, const W4Mat &w, const void *src, int dt, const float *scale, int br, int bc)
{
    // the pieces cover the codes' and the scales' padding too, so that no byte of either is left undefined
    const int lanes_log = w.cols <= 128 ? 2 : w.cols <= 256 ? 3 : w.cols <= 512 ? 4 : 5;
    const unsigned pieces = lanes_log < 5 ? 1 : (max(w.pitch * 2, w.sp * w.group) + CV_COLS - 1) / CV_COLS;
    const long long units = (w.rows + (32 >> lanes_log) - 1ll) / (32 >> lanes_log) * pieces;
    const int size = dt == DT_F32 ? 4 : dt == DT_BF16 ? 2 : 1;
    const size_t align = dt == DT_FP8 ? 8 : 16;
    const bool whole = (reinterpret_cast<uintptr_t>(src) % align) == 0 && ((size_t)w.cols * size) % align == 0;
    uint8_t *codes = const_cast<uint8_t *>(w.codes);
    uint16_t *scales = const_cast<uint16_t *>(w.scales);
    const int grid = (int)((units + CV_WARPS - 1) / CV_WARPS), scols = bc > 0 ? (w.cols + bc - 1) / bc : 0;
    const bool narrow = lanes_log < 5;
#define QUANTIZE_AS(DT, W, N) G5B_LAUNCH((w4_quantize_kernel<DT, W, N>), grid, CV_WARPS * 32, 0, st, w, codes, scales, src, scale, br, bc, scols, pieces, lanes_log)
#define QUANTIZE(DT)                                                                  \
    do {                                                                              \
        if (whole) { if (narrow) QUANTIZE_AS(DT, true, true); else QUANTIZE_AS(DT, true, false); }    \
        else       { if (narrow) QUANTIZE_AS(DT, false, true); else QUANTIZE_AS(DT, false, false); }  \
    } while (0)
    if (dt == DT_F32)       QUANTIZE(DT_F32);
    else if (dt == DT_BF16) QUANTIZE(DT_BF16);
    else                    QUANTIZE(DT_FP8);
#undef QUANTIZE
#undef QUANTIZE_AS
}

// A lane takes four columns at a time, so that a warp's store is 512 contiguous bytes of FP32 (eight columns a lane: 52 us for 12288 x 4096); of
// rows that do not allow that one column, the next lane the next (6319 x 2649 there and back 45 us in F32, 37 in BF16).
template <int DT>
__global__ void __launch_bounds__(CV_WARPS * 32) w4_dequantize_kernel(W4Mat w, void *out, size_t ldo, unsigned pieces, bool whole)
{
    const int lane = threadIdx.x & 31;
    const unsigned unit = blockIdx.x * CV_WARPS + (threadIdx.x >> 5), row_ = unit / pieces;
    const int row = (int)row_, c_first = (int)(unit - row_ * pieces) * CV_COLS + lane * 4, log = w.group == 128 ? 7 : w.group == 64 ? 6 : 5;
    if (row >= w.rows) return;
    if (!whole) {
        // a lane's word holds the codes of eight columns and goes round by shuffles; 32 columns have one scale
        const int p0 = c_first - lane * 4, words = w.pitch / 4 - p0 / 8;
        const uint32_t *codes = reinterpret_cast<const uint32_t *>(w.codes + (size_t)row * w.pitch) + p0 / 8;
        uint32_t word[CV_COLS / 256];
        float scale[CV_COLS / 256];
#pragma unroll
        for (int q = 0; q < CV_COLS / 256; q++) {
            const int c = p0 + q * 256 + (lane & 7) * 32;
            word[q] = q * 32 + lane < words ? __ldg(codes + q * 32 + lane) : 0u;
            scale[q] = c < w.cols ? bf16_to_f32(__ldg(w.scales + (size_t)row * w.sp + (c >> log))) : 0.f;
        }
#pragma unroll
        for (int q = 0; q < CV_COLS / 256; q++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int c = p0 + q * 256 + k * 32 + lane;
                if (c - lane >= w.cols) break;
                const uint32_t from = __shfl_sync(0xffffffffu, word[q], 4 * k + (lane >> 3));
                const float s = __shfl_sync(0xffffffffu, scale[q], k), v = __fmul_rn((float)((int)((from >> (4 * (lane & 7))) & 15u) - 8), s);
                if (c >= w.cols) continue;
                if (DT == DT_F32) __stcs(static_cast<float *>(out) + (size_t)row * ldo + c, v);
                else static_cast<__nv_bfloat16 *>(out)[(size_t)row * ldo + c] = __float2bfloat16_rn(v);
            }
        return;
    }
    uint32_t code[CV_COLS / 128];
    float s[CV_COLS / 128];
#pragma unroll
    for (int i = 0; i < CV_COLS / 128; i++) {
        const int c0 = c_first + 128 * i;
        code[i] = 0; s[i] = 0.f;
        if (c0 < w.cols) {
            code[i] = __ldg(reinterpret_cast<const uint16_t *>(w.codes + (size_t)row * w.pitch) + c0 / 4);
            s[i] = bf16_to_f32(__ldg(w.scales + (size_t)row * w.sp + (c0 >> log)));
        }
    }
#pragma unroll
    for (int i = 0; i < CV_COLS / 128; i++) {
        const int c0 = c_first + 128 * i;
        if (c0 >= w.cols) continue;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = __fmul_rn((float)((int)((code[i] >> (4 * k)) & 15u) - 8), s[i]);
        const size_t at = (size_t)row * ldo + c0;
        if (DT == DT_F32) {
            float *o = static_cast<float *>(out) + at;
            if (c0 + 4 <= w.cols) __stcs(reinterpret_cast<float4 *>(o), make_float4(v[0], v[1], v[2], v[3]));
            else
                for (int k = 0; k < 4 && c0 + k < w.cols; k++) o[k] = v[k];
        } else {
            // (3 significant bits times 8: rounded to BF16's 8, halves to even)
            __nv_bfloat16 *o = static_cast<__nv_bfloat16 *>(out) + at;
            if (c0 + 4 <= w.cols) {
                __align__(8) const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
                __stcs(reinterpret_cast<uint2 *>(o), *reinterpret_cast<const uint2 *>(h));
            } else
                for (int k = 0; k < 4 && c0 + k < w.cols; k++) o[k] = __float2bfloat16_rn(v[k]);
        }
    }
}

void w4_dequantize(cudaStream_t st, const W4Mat &w, void *out, int dt, size_t ldo)
{
    const unsigned pieces = (w.cols + CV_COLS - 1) / CV_COLS;
    const int size = dt == DT_F32 ? 4 : 2;
    const long long units = (long long)w.rows * pieces;
    const int grid = (int)((units + CV_WARPS - 1) / CV_WARPS);
    const bool whole = (reinterpret_cast<uintptr_t>(out) % (4 * size)) == 0 && ldo % 4 == 0;
    if (dt == DT_F32) G5B_LAUNCH(w4_dequantize_kernel<DT_F32>, grid, CV_WARPS * 32, 0, st, w, out, ldo, pieces, whole);
    else              G5B_LAUNCH(w4_dequantize_kernel<DT_BF16>, grid, CV_WARPS * 32, 0, st, w, out, ldo, pieces, whole);
}

}  // namespace g5b
