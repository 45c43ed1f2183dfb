// w4_many.cu - 4-bit weights times many activation rows (a batch, a prompt, an expert's share of one) on the tensor
// cores of sm_100: tcgen05.mma with the weights as the A operand out of tensor memory.
//
// A tile is two blocks of 128 weight rows (gate/up: 128 gate rows and the 128 up rows that go with them) and up to 64
// activation rows. One CTA per SM walks tiles; its warps have roles:
//   codes by TMA: 2 x 128 rows x 64 bytes (128 columns) a step
//   activation terms by TMA: 64 rows x 128 columns x terms a step
//   conversion, four warps to a block, a thread to a row: nibbles become F16 values of (code - 8) * scale in tensor
//          memory. They are exact: 3 significant bits of the code times 8 of a BF16 scale fit F16's 11, with a power of two per row
//          of W and step. A masked nibble is the subnormal number code * 2^-24 (or 2^-20), and one fused operation makes it
//          (code - 8) * scale while the step's scales are within 2^8 of each other: the largest times 2^24 lies below 2^16, the
//          smallest's products above F16's last bit. Otherwise 1024 + code, minus 1032, times the scale, whose largest is brought below
//          2^12: two operations, exact over 2^28 (groups of 32, eight rows past 154880 x 4096: 132 us).
//          (A power of two for a whole row needs all its scales before the first product: 7000 cycles a tile in groups of 32.)
//          Groups of 128: the codes alone (times 2^-17), and the scale on a step's sums.
//   products, one warp to a block: D[128 rows of W][rows of x] += A * terms^T; the two terms of an F32 row go into the
//          same sums, so that a converted block is used twice: a step's lower terms all before its upper ones, because each instruction cuts
//          what it adds to (products 2.5e-7 off 64 bits with the terms in turn, 1.0e-7 so; groups of 64 3.5e-7 and 1.8e-7).
//   sums, four warps to a block: take a step's sums out of tensor memory, take the power of two off (groups of 128: put the
//          scale on) and add them in registers, because the tensor cores cut off when they add; two accumulators in turn.
//          Sums in registers are 2^-35 of what they stand for: rows of x below 2^14 past 2^17 columns of codes below 2^3 and a finite scale
//          stay within FP32. At a tile's end that and the rows' powers of two come off, and the rows are stored. (At the other end a product is
//          off by 2^-128 of its row's largest activation.)
// BF16 rows have one term, a converted block is used once, and the conversion is most of a step: two groups of warps take steps in turn (2048
// rows past 12288 x 4096 288 -> 226 us; of F32 rows, whose sums then lack registers, 300 -> 327).
// A converted block and its sums live in tensor memory (256 columns each); shared memory only holds what TMA brings, which it
// must read for every product anyway: 64 rows of terms, 16 KB per step and term.
//
// A dense product's tiles are dealt out in rounds, whole; those of a last round that would leave SMs idle are cut along the columns, into
// parts whose sums a second kernel adds in order (605 tiles are 4 rounds of 148 and 13 tiles, which are cut into eleven). Equal shares of all
// steps instead, whatever the tiles, gave every CTA two tiles' beginnings and ends: 64 rows past 12288 x 4096 30.4 us against 27.3.
// Every wait is bounded: one that runs out sets a flag (g5b_w4_status), and every role drains what it has in flight and ends.
#include <algorithm>

#include "tc_ptx.cuh"
#include "w4.cuh"

namespace g5b {

constexpr int WM_ROWS = 64;                         // activation rows of a tile
// Groups of warps that convert, stages of codes (with two groups an even number, so that each stage belongs to one of them, and none of
// their waits can take another use's phase for its own) and of terms. Registers of a thread: what the launch gives all of them, and what
// those that hold the sums, convert and wait have of it then (256 * 120 + 384 * 80 = 640 * 96; 256 * 104 + 512 * 56 + 128 * 72 = 896 * 72).
template <int TERMS> struct ManyRoles;
template <> struct ManyRoles<2> { static constexpr int GROUPS = 1, WS = 3, XS = 3, SUM = 120, CONVERT = 80, REST = 80; };
template <> struct ManyRoles<1> { static constexpr int GROUPS = 2, WS = 4, XS = 3, SUM = 104, CONVERT = 56, REST = 72; };
template <int TERMS> constexpr int many_threads() { return (8 + 8 * ManyRoles<TERMS>::GROUPS + 4) * 32; }
constexpr int WM_W_STAGE = 2 * 128 * 64;
constexpr int WM_RING = 8;                          // steps whose powers of two are kept (the conversion is two stages and two accumulators ahead of the sums)
constexpr int WM_CTAS = 148;                        // SMs of a B200: what the cuts are chosen for
constexpr int WM_PARTS = 16;

static __device__ int g_many_err;                     // a wait that ran out: its code (0: none)

struct ManyMaps { CUtensorMap w, up, x; };
struct ManyArgs {
    W4Mat w, up;
    const float *inv;
    int mode, KB, n;               // steps of 128 columns; rows of a box of terms (a multiple of 16)
    int RT, TT;                    // tiles of weight rows; dense: tiles of activation rows
    int whole, parts;              // dense: tiles that are not cut, parts of the others
    int T;
    W4Slots slots;
    void *y;
    size_t ldy;
    int y_dt;
    float *part;                   // dense: sums of the tiles that are cut, [tile][part][n][256]
    int wide;                      // four rows of an output may be stored at once
    float limit;
};

struct ManyTile {
    int e, rt, first, np, n, k0, k1;
    int part;              // -1: the tile is not cut; else the place of its sums
};
// A CTA's work: items u, u + grid, ... (dense: whole tiles, then the others' parts; experts: tiles).
struct ManyWalk { int u, end; };
__device__ __forceinline__ ManyWalk many_walk(const ManyArgs &a)
{
    return ManyWalk{(int)blockIdx.x, a.mode == W4_DENSE ? a.whole + (a.RT * a.TT - a.whole) * a.parts : a.RT * load_new(a.slots.n)};
}
__device__ __forceinline__ bool many_next(const ManyArgs &a, ManyWalk &w, ManyTile &t)
{
    if (w.u >= w.end) return false;
    t.part = -1; t.k0 = 0; t.k1 = a.KB;
    if (a.mode == W4_DENSE) {
        int tile = w.u;
        if (tile >= a.whole) {
            // the same part of all tiles, then the next
            const int cut = a.RT * a.TT - a.whole, i = w.u - a.whole, q = i / cut, c = i - q * cut;
            tile = a.whole + c;
            t.k0 = a.KB * q / a.parts; t.k1 = a.KB * (q + 1) / a.parts;
            if (a.parts > 1) t.part = c * a.parts + q;
        }
        const int tt = tile % a.TT;
        t.e = 0; t.rt = tile / a.TT;
        t.first = tt * a.n; t.np = min(a.n, a.T - t.first);
    } else {
        const int slot = w.u / a.RT;
        t.rt = w.u - slot * a.RT;
        t.e = load_new(a.slots.expert + slot); t.first = load_new(a.slots.first + slot); t.np = load_new(a.slots.count + slot);
    }
    t.n = (t.np + 15) & ~15;
    w.u += gridDim.x;
    return true;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127

__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<uint32_t *>(&v); }
// Eight codes of a word as four pairs in the terms' order: (code - 8) 2^-17 (WHOLE: half of the 2^-35 that sums are held in, for nothing; subnormal
// F16 numbers are as exact as others), or times the scale (twice in s). That a nibble in the low bits of 1024 is the number 1024 + nibble, and in
// those of 2^-7 2^-7 + nibble 2^-17, is the usual way of taking such codes to F16. (A multiplication by 2^-17 instead: 64 rows 21 -> 22.6 us.)
template <bool WHOLE>
__device__ __forceinline__ void many_convert(uint32_t v, __half2 s, uint32_t *f)
{
    constexpr uint32_t BASE = WHOLE ? 0x20002000u : 0x64006400u;
    constexpr float P = WHOLE ? 0x1p-17f : 1.0f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t a, b;
        asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(a) : "r"(v), "n"(BASE));       // (v & mask) | base
        asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(b) : "r"(v), "n"(BASE));
        const __half2 lo = __hadd2(*reinterpret_cast<__half2 *>(&a), __float2half2_rn(-1032.f * P));
        const __half2 hi = __hfma2(*reinterpret_cast<__half2 *>(&b), __float2half2_rn(0.0625f), __float2half2_rn(-72.f * P));
        f[2 * i] = h2_bits(WHOLE ? lo : __hmul2(lo, s));
        f[2 * i + 1] = h2_bits(WHOLE ? hi : __hmul2(hi, s));
        v >>= 8;
    }
}
// The same from subnormal numbers. lo: the scale times 2^24; hi: times 2^20; off: times -8.
__device__ __forceinline__ void many_convert_fused(uint32_t v, __half2 lo, __half2 hi, __half2 off, uint32_t *f)
{
#pragma unroll
    for (int i = 0; i < 2; i++) {
        uint32_t a = v & 0x000f000fu, b = v & 0x00f000f0u;
        f[2 * i] = h2_bits(__hfma2(*reinterpret_cast<__half2 *>(&a), lo, off));
        f[2 * i + 1] = h2_bits(__hfma2(*reinterpret_cast<__half2 *>(&b), hi, off));
        v >>= 8;
    }
}

// Bounded wait for two or three barriers, looked at together: each look takes some 200 cycles even when the phase is long over, one after
// the other they were most of a step. The first, which is expected to be the last to come, is waited for without polling. By one thread, or by a whole warp in step (WARP).
template <bool WARP = false>
__device__ __forceinline__ bool many_wait(uint64_t *p, uint32_t pp, uint64_t *q, uint32_t qp, uint64_t *r, uint32_t rp, int *err, int code)
{
#pragma unroll 1
    for (int i = 0; i < ST_WAIT_LIMIT; i++) {
        const bool b = !q || mbar_test(q, qp), c = !r || mbar_test(r, rp), a = mbar_try_wait(p, pp);
        if (WARP ? __all_sync(0xffffffffu, a && b && c) : a && b && c) return true;
    }
    if (!WARP || (threadIdx.x & 31) == 0) atomicExch(err, code);
    if (WARP) __syncwarp();
    return false;
}

// True when it is true for all `threads` of a barrier: they go on together or not at all.
__device__ __forceinline__ bool many_all(bool ok, int barrier, int threads)
{
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((uint32_t)ok), "r"(barrier), "r"(threads) : "memory");
    return all != 0;
}

template <int TERMS, bool GATEUP, bool WHOLE>
__global__ void __launch_bounds__(many_threads<TERMS>(), 1) w4_many_kernel(const __grid_constant__ ManyMaps maps, const ManyArgs a)
{
    using Roles = ManyRoles<TERMS>;
    constexpr int WS = Roles::WS, XS = Roles::XS, GROUPS = Roles::GROUPS, REST = 8 + 8 * GROUPS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int XB = 2 * TERMS * a.n * 128;
    uint8_t *wst = smem;                                                     // [WS][2][128 rows][64]
    uint8_t *xst = wst + WS * WM_W_STAGE;                                 // [XS][64-column half][term][n rows][128]
    float *exch = reinterpret_cast<float *>(xst + (size_t)XS * XB);       // [block][64][128]
    __shared__ uint64_t w_full[WS], w_empty[WS], x_full[XS], x_empty[XS];
    __shared__ uint64_t a_full[2][2], a_empty[2][2], d_full[2][2], d_empty[2][2], drained[2];     // [block][stage]
    __shared__ uint32_t s_tmem;
    __shared__ float s_down[WM_RING][2][128];               // what takes a row's power of two off again
    int *err = &g_many_err;

    if (threadIdx.x == 0) {
        for (int i = 0; i < WS; i++) { mbar_init(&w_full[i], 1); mbar_init(&w_empty[i], 8); }
        for (int i = 0; i < XS; i++) { mbar_init(&x_full[i], 1); mbar_init(&x_empty[i], 2); }
        for (int b = 0; b < 2; b++) {
            for (int i = 0; i < 2; i++) { mbar_init(&a_full[b][i], 4); mbar_init(&a_empty[b][i], 1); mbar_init(&d_full[b][i], 1); mbar_init(&d_empty[b][i], 4); }
            mbar_init(&drained[b], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == REST + 2) tmem_alloc(&s_tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();                                          // (only now: whatever starts early may want tensor memory of its own, and this kernel has it)
    const uint32_t tmem = s_tmem;
    // sums of block b, accumulator i: columns 128 b + 64 i; converted block b of stage s: columns 256 + 128 s + 64 b
    if (a.mode != W4_DENSE) pdl_wait();                     // (the slots are another kernel's)
    ManyWalk walk = many_walk(a);
    ManyTile t;
    bool ok = true;

    // (the four warps of a group change their registers in one place)
    if (warp >= REST) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Roles::REST));
        if (warp == REST) {
            // --------------------------------------------------------------------- codes ----
            if (elect_one()) {
                int s = 0, ph = 1, issued = 0;
#pragma unroll 1
                while (ok && many_next(a, walk, t)) {
#pragma unroll 1
                    for (int kb = t.k0; kb < t.k1; kb++) {
                        if (issued >= WS && !(ok = mbar_wait(&w_empty[s], (uint32_t)ph, err, 1))) break;
                        mbar_expect_tx(&w_full[s], WM_W_STAGE);
                        uint8_t *dst = wst + (size_t)s * WM_W_STAGE;
                        if (GATEUP) {
                            tma_load_3d(dst, &maps.w, kb * 64, t.rt * 128, t.e, &w_full[s]);
                            tma_load_3d(dst + WM_W_STAGE / 2, &maps.up, kb * 64, t.rt * 128, t.e, &w_full[s]);
                        } else {
                            tma_load_3d(dst, &maps.w, kb * 64, t.rt * 256, t.e, &w_full[s]);
                            tma_load_3d(dst + WM_W_STAGE / 2, &maps.w, kb * 64, t.rt * 256 + 128, t.e, &w_full[s]);
                        }
                        issued++;
                        if (++s == WS) { s = 0; ph ^= 1; }
                    }
                }
                // copies in flight must land before shared memory goes away
                for (int j = issued - 1; j >= 0 && j >= issued - WS; j--) mbar_wait(&w_full[j % WS], (uint32_t)(j / WS) & 1, err, 2);
            }
            __syncwarp();
        } else if (warp == REST + 1) {
            // --------------------------------------------------------------------- terms ----
            pdl_wait();
            if (elect_one()) {
                int s = 0, ph = 1, issued = 0;
#pragma unroll 1
                while (ok && many_next(a, walk, t)) {
#pragma unroll 1
                    for (int kb = t.k0; kb < t.k1; kb++) {
                        if (issued >= XS && !(ok = mbar_wait(&x_empty[s], (uint32_t)ph, err, 3))) break;
                        mbar_expect_tx(&x_full[s], (uint32_t)XB);
                        tma_load_4d(xst + (size_t)s * XB, &maps.x, 0, t.first, 0, kb * 2, &x_full[s]);
                        issued++;
                        if (++s == XS) { s = 0; ph ^= 1; }
                    }
                }
                for (int j = issued - 1; j >= 0 && j >= issued - XS; j--) mbar_wait(&x_full[j % XS], (uint32_t)(j / XS) & 1, err, 4);
            }
            __syncwarp();
        } else {
            // ------------------------------------------------------------------ products ----
            if (elect_one()) {
                // (One warp for both blocks' products waited and issued for 2000 cycles a step, of which the tensor cores work 1184.)
                const int b = warp - REST - 2;
                int as = 0, ap = 0, xs = 0, xp = 0, steps = 0;
#pragma unroll 1
                while (ok && many_next(a, walk, t)) {
                    const uint32_t idesc = tc_idesc(0, t.n);
#pragma unroll 1
                    for (int kb = t.k0; kb < t.k1; kb++) {
                        const int buf = steps & 1;
                        if (!(ok = many_wait(&a_full[b][as], (uint32_t)ap, &x_full[xs], (uint32_t)xp, steps >= 2 ? &d_empty[b][buf] : nullptr, (uint32_t)((steps >> 1) - 1) & 1, err, 5))) break;
                        tc_fence_after();
                        const uint32_t d = tmem + (uint32_t)(b * 128 + buf * 64), ab = tmem + 256u + (uint32_t)(as * 128 + b * 64);
                        const uint32_t xb = smem_u32(xst) + (uint32_t)(xs * XB);
#pragma unroll
                        for (int m = TERMS - 1; m >= 0; m--)
#pragma unroll
                            for (int k = 0; k < 8; k++) {
                                const uint64_t bd = tc_smem_desc(xb + (uint32_t)(((k >> 2) * TERMS + m) * a.n * 128)) + 2 * (k & 3);
                                tc_mma_f16_ts(d, ab + (uint32_t)(k * 8), bd, idesc, k || m != TERMS - 1 ? 1u : 0u);
                            }
                        tc_commit(&a_empty[b][as]);
                        tc_commit(&x_empty[xs]);
                        tc_commit(&d_full[b][buf]);
                        steps++;
                        if (++as == 2) { as = 0; ap ^= 1; }
                        if (++xs == XS) { xs = 0; xp ^= 1; }
                    }
                }
                // nothing of this thread is in flight, and no arrival still to come, when the CTA ends
                tc_commit(&drained[b]);
                mbar_wait(&drained[b], 0, err, 8);
            }
            __syncwarp();
        }
    } else if (warp >= 8) {
        // --------------------------------------------------- codes -> F16 in tensor memory ----
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Roles::CONVERT));
        // A step's parity (of all tiles' in a row) is the stage that it is converted to; two groups take one each.
        const int group = GROUPS == 2 ? ((warp - 8) >> 2) & 1 : 0, b = GROUPS == 2 ? (warp - 8) >> 3 : (warp - 8) >> 2, quarter = warp & 3, r = quarter * 32 + lane, x = (r >> 1) & 3;
        const uint32_t dst = tmem + ((uint32_t)(quarter * 32) << 16) + 256u + (uint32_t)(b * 64);
        const int per = a.w.group == 128 ? 2 : a.w.group == 64 ? 1 : 0;        // a 32-column piece's group: piece >> per
        int steps = 0;                                                          // before the tile
#pragma unroll 1
        while (ok && many_next(a, walk, t)) {
            const W4Mat &w = GATEUP && b ? a.up : a.w;
            const int row = GATEUP ? t.rt * 128 + r : t.rt * 256 + b * 128 + r;
            const uint16_t *srow = w.scales + (size_t)t.e * a.w.scales_stride + (size_t)min(row, a.w.rows - 1) * a.w.sp;
            // Raw scales of a step's four pieces (the four that they are among), two steps ahead: one load whatever the group's size, because
            // what comes out of branches is put together behind them, and waits there.
            auto first_of = [&](int kb) { return (4 * min(kb, t.k1 - 1) >> per) & ~3; };
            auto fetch = [&](int kb) { return WHOLE ? make_uint2(0u, 0u) : __ldg(reinterpret_cast<const uint2 *>(srow + first_of(kb))); };
            int kb = t.k0 + (GROUPS == 2 ? (steps ^ group) & 1 : 0);
            uint2 next = fetch(kb), next1 = GROUPS == 1 ? fetch(kb + 1) : make_uint2(0u, 0u);
            auto convert = [&](int kb, uint2 &next) {
                const int step = steps + kb - t.k0, ws = step % WS, as = step & 1;
                __half2 s2[4];
                bool fused = false;
                if (!WHOLE) {
                    uint2 sc = next;
                    next = fetch(kb + 2);
                    // (a group behind the last: zero, whatever lies there)
                    const int last = a.w.groups - first_of(kb);              // of the four, how many are groups
                    if (last < 4) {
                        sc.x &= last > 1 ? 0xffffffffu : 0xffffu;
                        sc.y &= last > 3 ? 0xffffffffu : last > 2 ? 0xffffu : 0u;
                    }
                    // exponents of the largest scale and the smallest that is not zero; far from FP32's ends, so that no power of two leaves it
                    const uint32_t x0 = sc.x & 0x7fff7fffu, y0 = sc.y & 0x7fff7fffu, m2 = __vmaxu2(x0, y0), l2 = __vminu2(__vsub2(x0, 0x00010001u), __vsub2(y0, 0x00010001u));
                    const int top = max((int)(max(m2 & 0xffffu, m2 >> 16) >> 7), 1), low = (int)((min(l2 & 0xffffu, l2 >> 16) + 1) >> 7);
                    fused = __all_sync(0xffffffffu, top - low <= 8 && top >= 40 && top <= 220);
                    // (2^114 takes the least scale's last bit to 2^-19, which F16 holds, and 2^-114 2^-35 is the least FP32 number)
                    const int e = fused ? 15 + 127 - top : min(11 + 127 - top, 114);
                    const float up = pow2(e);
                    s_down[step & (WM_RING - 1)][b][r] = (fused ? pow2(24 - e) : pow2(-e)) * 0x1p-35f;
#pragma unroll
                    for (int piece = 0; piece < 4; piece++) {
                        const int g = (4 * kb + piece) >> per;
                        const uint32_t raw = (g & 2 ? sc.y : sc.x) >> (g & 1 ? 16 : 0);
                        s2[piece] = __float2half2_rn(bf16_to_f32((uint16_t)raw) * up);
                    }
                }
                uint64_t *full = &w_full[ws], *free_ = &a_empty[b][as];
                const uint32_t full_parity = (uint32_t)(step / WS) & 1;
                if (!(ok = many_wait<true>(step >= 2 ? free_ : full, step >= 2 ? (uint32_t)((step >> 1) - 1) & 1 : full_parity, full, full_parity, nullptr, 0u, err, 9))) return;
                tc_fence_after();
                const uint8_t *src = wst + (size_t)ws * WM_W_STAGE + b * (WM_W_STAGE / 2) + r * 64;
                if (!WHOLE && fused) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t f[32];
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const int piece = h * 2 + c;
                            const __half2 hi = __hmul2(s2[piece], __float2half2_rn(0.0625f)), off = __hmul2(s2[piece], __float2half2_rn(-0x1p-21f));
                            const uint4 q = *reinterpret_cast<const uint4 *>(src + ((piece ^ x) << 4));
                            many_convert_fused(q.x, s2[piece], hi, off, f + c * 16); many_convert_fused(q.y, s2[piece], hi, off, f + c * 16 + 4);
                            many_convert_fused(q.z, s2[piece], hi, off, f + c * 16 + 8); many_convert_fused(q.w, s2[piece], hi, off, f + c * 16 + 12);
                        }
                        tmem_st32(dst + (uint32_t)(as * 128 + h * 32), f);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        uint32_t f[32];
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const int piece = h * 2 + c;
                            const uint4 q = *reinterpret_cast<const uint4 *>(src + ((piece ^ x) << 4));
                            many_convert<WHOLE>(q.x, s2[piece], f + c * 16); many_convert<WHOLE>(q.y, s2[piece], f + c * 16 + 4);
                            many_convert<WHOLE>(q.z, s2[piece], f + c * 16 + 8); many_convert<WHOLE>(q.w, s2[piece], f + c * 16 + 12);
                        }
                        tmem_st32(dst + (uint32_t)(as * 128 + h * 32), f);
                    }
                }
                // (handed back only here: the loads' values have arrived when they have been used)
                __syncwarp();
                if (lane == 0) mbar_arrive(&w_empty[ws]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_full[b][as]);
            };
            // (two sets of registers for the scales that are on their way: moved from one to the other they would be waited for)
#pragma unroll 1
            for (; kb < t.k1 && ok; kb += 2) {
                convert(kb, next);
                if (GROUPS == 1 && ok && kb + 1 < t.k1) convert(kb + 1, next1);
            }
            steps += t.k1 - t.k0;
        }
    } else {
        // ------------------------------------------------------------ sums, scales, stores ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Roles::SUM));
        const int b = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * 128);
        const int bar = GATEUP ? 1 : 1 + b, bar_threads = GATEUP ? 256 : 128;       // (gate/up: both blocks together)
        int steps = 0;
        pdl_wait();
#pragma unroll 1
        while (many_next(a, walk, t)) {
            // what the rows' finished sums are multiplied by: 2^35 and their powers of two, 2^-126 to 2^114
            float i0 = (lane < t.np ? load_new(a.inv + t.first + lane) : 0.f) * 0x1p35f, i1 = (lane + 32 < t.np ? load_new(a.inv + t.first + lane + 32) : 0.f) * 0x1p35f;
            F2 acc[WM_ROWS / 2];
#pragma unroll
            for (int k = 0; k < WM_ROWS / 2; k++) acc[k] = f2(0.f, 0.f);
            // what a step's sums are multiplied by: a step's scale, one step ahead (WHOLE), or what takes the power of two off
            const W4Mat &w = GATEUP && b ? a.up : a.w;
            const int row = GATEUP ? t.rt * 128 + r : t.rt * 256 + b * 128 + r;
            const uint16_t *srow = w.scales + (size_t)t.e * a.w.scales_stride + (size_t)min(row, a.w.rows - 1) * a.w.sp;
            uint16_t next = 0;
            if (WHOLE) next = __ldg(srow + t.k0);
#pragma unroll 1
            for (int kb = t.k0; kb < t.k1; kb++, steps++) {
                const int buf = steps & 1;
                float sc = bf16_to_f32(next) * 0x1p-18f;
                if (WHOLE && kb + 1 < t.k1) next = __ldg(srow + kb + 1);
                if (!(ok = mbar_wait_all(&d_full[b][buf], (uint32_t)(steps >> 1) & 1, err, 11))) break;
                if (!WHOLE) sc = s_down[steps & (WM_RING - 1)][b][r];
                tc_fence_after();
#pragma unroll
                for (int g = 0; g < WM_ROWS; g += 32)
                    if (g < t.n) {                                     // (columns past the rows hold nothing that is stored)
                        uint32_t v[2][16];
                        tmem_ld16(lane_addr + (uint32_t)(buf * 64 + g), v[0]);
                        tmem_ld16(lane_addr + (uint32_t)(buf * 64 + g + 16), v[1]);
                        tmem_ld_wait();
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            const F2 in = f2(__uint_as_float(v[k >> 3][2 * (k & 7)]), __uint_as_float(v[k >> 3][2 * (k & 7) + 1]));
                            acc[g / 2 + k] = f2_fma(in, f2(sc, sc), acc[g / 2 + k]);
                        }
                    }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&d_empty[b][buf]);
            }
            if (!(ok = many_all(ok, bar, bar_threads))) break;
            // Through shared memory, so that what comes now is a loop (unrolled over the registers it was 38000 cycles of a cold
            // instruction cache per tile) in which a warp stores 128 weight rows of one activation row, four to a lane.
            float *sums = exch + b * (WM_ROWS * 128);
#pragma unroll
            for (int k = 0; k < WM_ROWS; k += 2) {
                float x, y;
                f2_get(acc[k / 2], x, y);
                sums[k * 128 + r] = x;
                sums[k * 128 + 128 + r] = y;
            }
            many_all(true, bar, bar_threads);
            const int row0 = (GATEUP ? t.rt * 128 : t.rt * 256 + b * 128) + lane * 4;
            if (__any_sync(0xffffffffu, isinf(i0) || isinf(i1))) {
                // (rows with activations from 2^106 on, whose factor FP32 does not hold: 2^35 goes into the sums here. Apart from the loop below,
                // in which every instruction counts: a second factor there was 2 % of 2048 rows past 12288 x 4096.)
#pragma unroll 1
                for (int k = GATEUP ? warp : quarter; k < t.np; k += GATEUP ? 8 : 4)
                    if (isinf(__shfl_sync(0xffffffffu, k < 32 ? i0 : i1, k & 31)))
#pragma unroll 1
                        for (int q = 0; q < 4; q++) {
                            float *at = (GATEUP ? exch : sums) + k * 128 + lane * 4 + q;
                            *at *= 0x1p35f;
                            if (GATEUP) at[WM_ROWS * 128] *= 0x1p35f;
                        }
                if (isinf(i0)) i0 = load_new(a.inv + t.first + lane);
                if (isinf(i1)) i1 = load_new(a.inv + t.first + lane + 32);
            }
#pragma unroll 1
            for (int k = GATEUP ? warp : quarter; k < t.np; k += GATEUP ? 8 : 4) {
                const float inv = __shfl_sync(0xffffffffu, k < 32 ? i0 : i1, k & 31);
                const float4 in = *reinterpret_cast<const float4 *>((GATEUP ? exch : sums) + k * 128 + lane * 4);
                float v[4] = {in.x * inv, in.y * inv, in.z * inv, in.w * inv};
                if (GATEUP) {
                    const float4 up = *reinterpret_cast<const float4 *>(exch + (WM_ROWS + k) * 128 + lane * 4);
                    const float u[4] = {up.x * inv, up.y * inv, up.z * inv, up.w * inv};
#pragma unroll
                    for (int q = 0; q < 4; q++) v[q] = swiglu_value(v[q], u[q], a.limit);
                }
                const size_t at = (size_t)(t.first + k) * a.ldy + row0;
                if (!GATEUP && t.part >= 0)
                    *reinterpret_cast<float4 *>(a.part + ((size_t)t.part * a.n + k) * 256 + b * 128 + lane * 4) = make_float4(v[0], v[1], v[2], v[3]);
                else if (a.y_dt == DT_F32) {
                    float *y = static_cast<float *>(a.y) + at;
                    if (a.wide && row0 + 3 < a.w.rows) *reinterpret_cast<float4 *>(y) = make_float4(v[0], v[1], v[2], v[3]);
                    else
#pragma unroll
                        for (int q = 0; q < 4; q++) if (row0 + q < a.w.rows) y[q] = v[q];
                } else {
                    __nv_bfloat16 *y = static_cast<__nv_bfloat16 *>(a.y) + at;
                    __align__(8) const __nv_bfloat162 h[2] = {__floats2bfloat162_rn(v[0], v[1]), __floats2bfloat162_rn(v[2], v[3])};
                    if (a.wide && row0 + 3 < a.w.rows) *reinterpret_cast<uint2 *>(y) = *reinterpret_cast<const uint2 *>(h);
                    else
#pragma unroll
                        for (int q = 0; q < 4; q++) if (row0 + q < a.w.rows) y[q] = __float2bfloat16_rn(v[q]);
                }
            }
            // the buffer is free again
            many_all(true, bar, bar_threads);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == REST + 2) { __syncwarp(); tmem_dealloc(tmem, 512); }
}

// The tiles that were cut: their parts' sums in order. A CTA takes four rows of x of one tile.
__global__ void __launch_bounds__(256) w4_parts_kernel(const float *part, int parts, int whole, int TT, int n, int T, int rows, void *y, size_t ldy, int y_dt, int wide)
{
    pdl_wait();
    const int tile = whole + blockIdx.x, tt = tile % TT, k = blockIdx.y * 4 + (threadIdx.x >> 6), r = (threadIdx.x & 63) * 4, row = tile / TT * 256 + r;
    if (k >= n || tt * n + k >= T || row >= rows) return;
    const float *p = part + ((size_t)blockIdx.x * parts * n + k) * 256 + r;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < parts; q++) {
        const float4 in = __ldcs(reinterpret_cast<const float4 *>(p + (size_t)q * n * 256));
        v.x += in.x; v.y += in.y; v.z += in.z; v.w += in.w;
    }
    const size_t at = (size_t)(tt * n + k) * ldy + row;
    const float o[4] = {v.x, v.y, v.z, v.w};
    if (wide && row + 3 < rows && y_dt == DT_F32) *reinterpret_cast<float4 *>(static_cast<float *>(y) + at) = v;
    else
#pragma unroll
        for (int q = 0; q < 4; q++)
            if (row + q < rows) {
                if (y_dt == DT_F32) static_cast<float *>(y)[at + q] = o[q];
                else static_cast<__nv_bfloat16 *>(y)[at + q] = __float2bfloat16_rn(o[q]);
            }
}

static int many_box(int T) { return T < WM_ROWS ? (T + 15) / 16 * 16 : WM_ROWS; }
// Which tiles of a dense product are cut, and into how many parts: what takes the fewest steps of 128 columns, where the beginning and end of
// an item count as three and the second kernel as two.
struct ManyCut { int whole, parts; };
static ManyCut many_cut(int rows, int cols, int T)
{
    const int KB = w4_kp(cols) / 128, tiles = (rows + 255) / 256 * ((T + many_box(T) - 1) / many_box(T)), rounds = tiles / WM_CTAS;
    ManyCut best{tiles, 1};
    long long least = 0;
    for (int r = rounds; r >= 0 && r >= rounds - 1; r--)
        for (int p = 1; p <= WM_PARTS && (p == 1 || KB / p >= 2); p++) {
            const long long left = tiles - (long long)r * WM_CTAS;
            const long long cost = r * (KB + 3ll) + (left * p + WM_CTAS - 1) / WM_CTAS * ((KB + p - 1) / p + 3) + (p > 1 ? 2 : 0);
            if ((r == rounds && p == 1) || cost < least) { least = cost; best = p > 1 ? ManyCut{r * WM_CTAS, p} : ManyCut{tiles, 1}; }
        }
    return best;
}
size_t w4_many_part_floats(int rows, int cols, int T)
{
    const ManyCut c = many_cut(rows, cols, T);
    const size_t tiles = (size_t)((rows + 255) / 256) * ((T + many_box(T) - 1) / many_box(T));
    return (tiles - c.whole) * c.parts * many_box(T) * 256;
}

template <int TERMS, bool GATEUP, bool WHOLE>
static int many_launch(cudaStream_t st, const ManyMaps &m, const ManyArgs &a, int grid)
{
    static SmemGrant grant;
    const size_t smem = 1024 + ManyRoles<TERMS>::WS * WM_W_STAGE + (size_t)ManyRoles<TERMS>::XS * 2 * TERMS * a.n * 128 + 2 * WM_ROWS * 128 * 4;
    if (!dev_opt_in_smem((const void *)w4_many_kernel<TERMS, GATEUP, WHOLE>, smem, grant)) return -1;
    G5B_LAUNCH_PDL((w4_many_kernel<TERMS, GATEUP, WHOLE>), dim3(grid), dim3(many_threads<TERMS>()), smem, st, m, a);
    return 0;
}

int w4_many(cudaStream_t st, const W4Job &j, float *part)
{
    ManyMaps m;
    ManyArgs a{};
    const int rows_most = j.mode == W4_DENSE ? j.T : j.slots.rows;
    a.w = j.w; a.up = j.up; a.inv = j.terms.inv; a.mode = j.mode; a.KB = j.terms.kp / 128; a.T = j.T; a.slots = j.slots;
    a.n = many_box(rows_most);
    a.RT = (j.w.rows + (j.mode == W4_GATEUP ? 127 : 255)) / (j.mode == W4_GATEUP ? 128 : 256);
    a.TT = (j.T + a.n - 1) / a.n;
    a.y = j.y; a.ldy = j.ldy; a.y_dt = j.y_dt; a.part = part; a.limit = j.limit;
    a.wide = j.ldy % 4 == 0 && reinterpret_cast<uintptr_t>(j.y) % (j.y_dt == DT_F32 ? 16 : 8) == 0;
    const cuuint64_t wsize[3] = {(cuuint64_t)j.w.pitch, (cuuint64_t)j.w.rows, (cuuint64_t)j.count};
    const cuuint64_t wstride[2] = {(cuuint64_t)j.w.pitch, (cuuint64_t)j.w.codes_stride};
    const cuuint32_t wbox[3] = {64, 128, 1};
    const cuuint64_t row = (cuuint64_t)j.terms.n_terms * j.terms.kp * 2;
    const cuuint64_t xsize[4] = {64, (cuuint64_t)j.T, (cuuint64_t)j.terms.n_terms, (cuuint64_t)j.terms.kp / 64}, xstride[3] = {row, (cuuint64_t)j.terms.kp * 2, 128};
    const cuuint32_t xbox[4] = {64, (cuuint32_t)a.n, (cuuint32_t)j.terms.n_terms, 2};
    if (!tc_encode_swizzled(&m.w, j.w.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, wsize, wstride, wbox, CU_TENSOR_MAP_SWIZZLE_64B) ||
        (j.mode == W4_GATEUP && !tc_encode_swizzled(&m.up, j.up.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, wsize, wstride, wbox, CU_TENSOR_MAP_SWIZZLE_64B)) ||
        !tc_encode_swizzled(&m.x, j.terms.terms, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, xsize, xstride, xbox, CU_TENSOR_MAP_SWIZZLE_128B)) {
        set_last_error("a tensor map of a 4-bit product was refused");
        return -1;
    }
    const int tiles = a.RT * a.TT;
    long long items = (long long)a.RT * j.slots.max;
    if (j.mode == W4_DENSE) {
        const ManyCut cut = many_cut(j.w.rows, j.w.cols, j.T);
        a.whole = cut.whole; a.parts = cut.parts;
        items = a.whole + (long long)(tiles - a.whole) * a.parts;
    }
    const int grid = (int)std::min<long long>(items, dev_sms());
    const bool pair = j.mode == W4_GATEUP, whole = j.w.group == 128;
    const int rc = j.terms.n_terms == 1 ? whole ? (pair ? many_launch<1, true, true>(st, m, a, grid) : many_launch<1, false, true>(st, m, a, grid))
                                                : (pair ? many_launch<1, true, false>(st, m, a, grid) : many_launch<1, false, false>(st, m, a, grid))
                                        : whole ? (pair ? many_launch<2, true, true>(st, m, a, grid) : many_launch<2, false, true>(st, m, a, grid))
                                                : (pair ? many_launch<2, true, false>(st, m, a, grid) : many_launch<2, false, false>(st, m, a, grid));
    if (rc) return -1;
    if (j.mode == W4_DENSE && a.parts > 1)
        G5B_LAUNCH_PDL(w4_parts_kernel, dim3(tiles - a.whole, (a.n + 3) / 4), dim3(256), 0, st, part, a.parts, a.whole, a.TT, a.n, j.T, j.w.rows, j.y, j.ldy, j.y_dt, a.wide);
    return 0;
}

int w4_many_status(cudaStream_t st) { return w4_flag(g_many_err, st); }

}  // namespace g5b
