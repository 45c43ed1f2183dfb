// w4_few.cu - 4-bit weights times a few rows of activations: a decoded token or two, the few tokens of an expert in a batch. Eight columns at
// a time: two rows of four digits, F32 or BF16. (Four rows in two sets of columns: an item of three or four rows takes 1.5 times as long as one of
// two, and CTAs that have such items end last. Experts of 64 tokens 831 us against 752.)
//
// Bound by HBM: half a byte and a scale's share per weight (154880 x 4096 past one row 54.3 us, 6.0 TB/s; a launch's start and end are 4 of them,
// and all of the 5 us that 4096 x 2048 takes). The integer matrix instruction does the products (16 weight rows x 32
// columns x 8 activation columns, twice the F16 one's): codes are the unsigned operand nearly as they are, where
// F16 values took five logical and four packed operations to eight of them; activations are 8-bit digits of a fixed-point number; sums are exact.
// One CTA per SM, persistent. Work comes in items of 16 weight rows (gate/up: eight gate rows and the eight up rows that go with them),
// in pieces of 4096 columns; a CTA takes a contiguous share of them. Of up to 2048 columns an item is 32 rows: with two blocks of 128
// columns to a warp its waits and the sums' meeting were most of an item (down products of 64 tokens' experts 282 us at 4.5 TB/s;
// all three products 736 -> 648 us in short runs, 32768 x 800 past two rows 12.9 -> 10.3).
//   warp 16   brings an item's rows into a ring in shared memory, one TMA load for the codes and one for the scales (gate/up: two
//             each), as many ahead as fit: they wait for nothing but room, so HBM is busy while sums are put together and rows change.
//             (A bulk copy per row was 125 cycles of issue each: 2.3 TB/s.)
//   0-7, 8-15 take items in turn, from rings of their own; the eight warps of a team share an item's blocks of 128 columns, and their sums meet in shared
//             memory in a fixed order
//   codes     a lane takes 16 bytes of rows g and g + 8 (lane = 4 g + t), a quad 64 bytes: 128 columns of each. Which column stands for
//             which k of an MMA does not matter as long as both operands agree, and the digits lie in that order. In groups of 128 a
//             byte is an operand as it is, 16 h + l, past the odd columns' digits o, and its low nibble another, past digits of
//             e - o / 16: l e + h o = (16 h + l) o / 16 + l (e - o / 16), one AND to eight codes. (High nibbles masked too, eight moves
//             and a multiplication of each scale: 770 us for the experts of 64 tokens at the power limit's 1.6 GHz, where instructions bound them.) What the codes' offset of
//             8 adds is known from the digits: the sums start at minus that.
//   scales    in FP32, once per group, on the sums of the group. A quad's 128 columns are one group of 128; for smaller groups
//             a lane takes its words 16 bytes apart, so that an MMA is 32 columns of one group.
//   x         becomes digits in shared memory whenever the rows change (dense: once; experts: with the expert), in the order in
//             which the lanes read them: per row and block of 128 columns the power of two below which its values lie, and
//             integers of 31 bits and a sign in four digits, one bit less where the largest needs it: an FP32 number down to 2^-6 of the block's largest and a
//             BF16 one down to 2^-22 as they are (in groups of 128 even columns are off by half a unit), what is smaller by a unit, 2^-29 of the largest, at most. (Three digits of F32 rows and two of BF16
//             ones, four of which then fit, were off by 2^-22 and 2^-14 of the largest: by 3e-5 and 8e-3 of a product whose weights of columns a
//             thousand times the others are small. The fourth digit takes a column that was idle.)
// Group sums are exact integers, taken into FP32 by the exponent trick: they start at the bits of 48, so that their bits are the float
// 48 + sum 2^-18, |sum| < 2^18 (in groups of 128 at those of 3, in sixteenths); sums across groups are FP32. Whatever the scales and
// activations, no intermediate leaves FP32's range where the sums of a result's magnitudes do not: sum 2^-18 < 1 times a scale, times
// a digit's worth 2^5 < 2^128, and 2^13 once an output's sums are complete. At the other end a product is off by 2^-139 of the largest activation, a sum by 2^-136. Every wait is bounded: one that runs out sets a flag (g5b_w4_status).
#include <algorithm>

#include "tc_ptx.cuh"
#include "w4.cuh"

namespace g5b {

constexpr int FW_WARPS = 16, FW_THREADS = (FW_WARPS + 1) * 32;
constexpr int FW_COLS = 8;                           // activation columns of an MMA
constexpr int FW_DIGITS = 4;                         // of an activation, a column each
constexpr int FW_ROWS = FW_COLS / FW_DIGITS;
constexpr int FW_PIECE = 4096;                       // weight columns of a stage at most (half of them where that leaves too few stages): 16 chunks of 128 bytes
constexpr int FW_DIGIT_BYTES = 88 * 1024;            // room for the digits
constexpr int FW_MAX_STAGES = 12;
constexpr int FW_SUMS = 16 * 1024;                   // sums of a sixteen of weight rows
constexpr int FW_SMEM = 206 * 1024;                  // for stages and digits with the sums of a sixteen beside them

static __device__ int g_few_err;                     // a wait that ran out: its code (0: none)

struct FewMaps { CUtensorMap codes[2], scales[2]; };  // gate/up: of either; else the first
struct FewArgs {
    W4Mat w;
    const void *x;
    size_t ldx;
    int x_dt, cols, blocks;        // columns of x, blocks of 128 of them
    int wide;                      // x may be read 16 bytes at a time
    int tiles, rows, per;          // row tiles; dense: rows of x; rows of a slot at most
    const int *order, *idx;        // experts: sorted picks, or (idx) the picks themselves, each a slot of its own
    int topk, E, n;
    W4Slots slots;
    void *y;
    size_t ldy;
    int y_dt;
    float limit;
    int whole_rows;                // rows of codes are whole chunks: one load brings all of a stage's
    int piece;                     // blocks of 128 columns of a stage
    int sixteens;                  // of weight rows of an item
    int chunks, scale_cols;        // of a stage at most
    int scale_pitch;               // scales of a stage's row: eight more, so that eight rows lie in different banks
    int stages, stage_bytes, stage_tx;      // (stages of a team)
};
struct FewItem { int e, first, count, tile; };       // expert; sorted rows (dense: rows of x); row tile
// here: picks of experts that are here (idx: a bit each)
template <int MODE>
__device__ __forceinline__ int few_slots(const FewArgs &a, uint32_t here) { return MODE == W4_DENSE ? 1 : a.idx ? __popc(here) : load_new(a.slots.n); }
template <int MODE>
__device__ __forceinline__ FewItem few_item(const FewArgs &a, uint32_t here, int slot, int tile)
{
    if (MODE == W4_DENSE) return FewItem{0, 0, a.rows, tile};
    if (a.idx) {
        for (int k = 0; k < slot; k++) here &= here - 1;
        const int pick = __ffs(here) - 1;
        return pick < 0 ? FewItem{} : FewItem{__ldg(a.idx + pick), pick, 1, tile};
    }
    return FewItem{load_new(a.slots.expert + slot), load_new(a.slots.first + slot), load_new(a.slots.count + slot), tile};
}

// (not volatile: two blocks' chains of these are put side by side)
__device__ __forceinline__ void few_mma(int (&c)[4], uint32_t g0, uint32_t h0, uint32_t g1, uint32_t h1, uint32_t b0, uint32_t b1, int s0, int s1, int s2, int s3)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(g0), "r"(h0), "r"(g1), "r"(h1), "r"(b0), "r"(b1), "r"(s0), "r"(s1), "r"(s2), "r"(s3));
}
__device__ __forceinline__ void few_mma(int (&c)[4], uint32_t g0, uint32_t h0, uint32_t g1, uint32_t h1, uint32_t b0, uint32_t b1)
{
    few_mma(c, g0, h0, g1, h1, b0, b1, c[0], c[1], c[2], c[3]);
}
__device__ __forceinline__ float few_pow2(int e) { return __int_as_float((e + 127) << 23); }      // -126 <= e <= 127
// The bits of 48, whose last is worth 2^-18, or for sums of sixteenths of 3.
template <bool WHOLE> constexpr int few_magic = WHOLE ? 0x40400000 : 0x42400000;
template <bool WHOLE> __device__ __forceinline__ float few_float(int v) { return __fsub_rn(__int_as_float(v), WHOLE ? 3.0f : 48.0f); }
constexpr float FW_REST = 8192.0f;                   // what is left of 2^18 when 2^5 are part of a digit's worth
__device__ __forceinline__ uint32_t word_of(const uint4 &v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// A block of 128 columns: [part][column][t] 16 bytes of digits as the lanes read them, then for each of the eight columns where the sums
// start (WHOLE: of the block; else of each 32 columns, with groups of 64 those of both halves in the first) and what a digit stands for, times 2^5.
template <int NS, bool WHOLE> struct FewBlock {
    uint4 digits[2][NS][4];
    int   start[WHOLE ? 1 : 4][FW_COLS];
    float worth[FW_COLS];
};

// The 512 consumer threads: rows of an item as digits; 16 lanes hold a block.
template <int MODE, bool WHOLE, int NS, typename IN>
__device__ __forceinline__ void few_digits(const FewArgs &a, const FewItem &it, FewBlock<NS, WHOLE> *blocks)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = it.count <= 1 ? 1 : FW_ROWS, per = FW_WARPS / rows;    // warps to a row
    const int i = warp / per;
    bar_sync(1, FW_WARPS * 32);                          // nobody reads the digits of the rows before any more
    if (i < it.count) {
        const int at = it.first + i;
        const int src = MODE != W4_GATEUP ? at : (a.idx ? at : load_new(a.order + at)) / a.topk;
        const IN *row = static_cast<const IN *>(a.x) + (size_t)src * a.ldx;
        const int col = i * FW_DIGITS;
        for (int c0 = (warp - i * per) * 256; c0 < a.blocks * 128; c0 += per * 256) {
            const int c = c0 + lane * 8;
            float v[8];
            w4_load8(v, row, c, a.cols, a.wide);
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const bool finite = m < 0x7f800000u;
            // 2^(e - 1) <= max < 2^e (a subnormal one counts as 2^-126). One more bit where the largest leaves the highest digit below 128. (A unit
            // is 2^-149 at least, the smallest FP32 number, of which all others are multiples.)
            const int e = max((int)(m >> 23), 1) - 126;
            constexpr float MOST = 127.0f * 16777216.0f + 127.0f * 65536.0f + 127.0f * 256.0f;
            const float largest = __uint_as_float(m) * few_pow2((31 - e) >> 1) * few_pow2(31 - e - ((31 - e) >> 1));
            const int up = min(30 - e + (largest * (WHOLE ? 1.0625f : 1.0f) <= MOST), 149);          // -98 <= up
            const float scale = few_pow2(up >> 1), scale2 = few_pow2(up - (up >> 1));
            int x[8];
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = finite ? __float2int_rn(v[k] * scale * scale2) : 0;
            if (WHOLE)                                   // (the odd columns' integers, so that what they are off goes with their own weights alone)
#pragma unroll
                for (int k = 0; k < 8; k += 2) x[k] -= (x[k + 1] + 8) >> 4;
            uint32_t even[FW_DIGITS] = {}, odd[FW_DIGITS] = {};  // digits of columns 0 2 4 6 and 1 3 5 7
            int sum[FW_DIGITS] = {};
#pragma unroll
            for (int k = 0; k < 8; k++) {
                int rest = x[k];
#pragma unroll
                for (int d = 0; d < FW_DIGITS; d++) {
                    const int digit = d + 1 < FW_DIGITS ? (int)(int8_t)rest : rest;
                    rest = (rest - digit) >> 8;
                    sum[d] += digit * (WHOLE ? (k & 1 ? 136 : 128) : 8);
                    (k & 1 ? odd : even)[d] |= (uint32_t)(digit & 255) << (8 * (k >> 1));
                }
            }
            FewBlock<NS, WHOLE> &b = blocks[min(c >> 7, a.blocks - 1)];
            const bool here = c < a.blocks * 128;
            const int w = (c & 127) >> 3, j = WHOLE ? w & 3 : w >> 2, t = WHOLE ? w >> 2 : w & 3;
            const int span = a.w.group == 128 ? 16 : a.w.group == 64 ? 8 : 4;          // lanes of a group
#pragma unroll
            for (int d = 0; d < FW_DIGITS; d++) {
                for (int o = 1; o < span; o <<= 1) sum[d] += __shfl_xor_sync(0xffffffffu, sum[d], o);
                if (!here) continue;
                if (WHOLE) {
                    reinterpret_cast<uint32_t *>(&b.digits[0][col + d][t])[j] = even[d];
                    reinterpret_cast<uint32_t *>(&b.digits[1][col + d][t])[j] = odd[d];
                    if (w == 0) b.start[0][col + d] = few_magic<WHOLE> - sum[d];
                } else {
                    reinterpret_cast<uint2 *>(&b.digits[j >> 1][col + d][t])[j & 1] = make_uint2(even[d], odd[d]);
                    if ((lane & (span - 1)) == 0) b.start[WHOLE ? 0 : j][col + d] = few_magic<WHOLE> - sum[d];
                }
                if (w == 0) b.worth[col + d] = finite ? few_pow2(5 - (up >> 1)) * few_pow2(8 * d - (up - (up >> 1))) : __int_as_float(0x7fc00000);
            }
        }
    }
    __syncwarp();
    bar_sync(1, FW_WARPS * 32);
}

// IN: of activations. WHOLE: groups of 128. NS: columns that there is room for. U: sixteens of weight rows of an item.
template <typename IN, int MODE, bool WHOLE, int NS, int U>
__global__ void __launch_bounds__(FW_THREADS, 1) w4_few_kernel(const __grid_constant__ FewMaps maps, const FewArgs a)
{
    constexpr int HALVES = MODE == W4_GATEUP ? 2 : 1, HALF_ROWS = 16 * U / HALVES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    uint8_t *ring = smem;                                                             // [team][stages][half][chunk][row][128] codes, [half][row][scale_pitch] scales
    using Block = FewBlock<NS, WHOLE>;
    Block *blocks = reinterpret_cast<Block *>(smem + (size_t)2 * a.stages * a.stage_bytes);
    // A team waits for every use of its stages, so none of its waits can take an earlier use's phase for the one it waits for.
    __shared__ uint64_t full[2][FW_MAX_STAGES], empty[2][FW_MAX_STAGES];
    __shared__ __align__(16) float s_sum[2][2][8][16 * U][FW_COLS];                                // [team][item's parity][warp][row][column]
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    int *err = &g_few_err;
    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; i++)
            for (int k = 0; k < 2; k++) { mbar_init(&full[k][i], 1); mbar_init(&empty[k][i], 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (MODE != W4_DENSE && !a.idx) pdl_wait();           // (the slots are another kernel's)
    const int pieces = (a.blocks + a.piece - 1) / a.piece;
    uint32_t here = 0;
    if (MODE != W4_DENSE && a.idx) {
        const int e = lane < a.n ? __ldg(a.idx + lane) : -1;
        here = __ballot_sync(0xffffffffu, e >= 0 && e < a.E);
    }
    const long long items = (long long)few_slots<MODE>(a, here) * a.tiles;
    const long long i0 = items * blockIdx.x / gridDim.x, i1 = items * (blockIdx.x + 1) / gridDim.x;
    bool ok = true;
    int turn = 0;                                         // the team that takes the item

    if (warp == FW_WARPS) {
        // ------------------------------------------------------------------- weights ----
        if (elect_one()) {
            int slot = (int)(i0 / a.tiles), tile = (int)(i0 - (long long)slot * a.tiles), stage[2] = {0, 0}, parity[2] = {1, 1}, issued[2] = {0, 0};
            FewItem it = i0 < i1 ? few_item<MODE>(a, here, slot, tile) : FewItem{};
#pragma unroll 1
            for (long long i = i0; i < i1 && ok; i++) {
                if (it.count) {
                    // (the parity that the stage's `empty` must have passed: that of the use before)
                    int &st = stage[turn];
#pragma unroll 1
                    for (int p = 0; p < pieces; p++) {
                        if (issued[turn] >= a.stages && !(ok = mbar_wait(&empty[turn][st], (uint32_t)parity[turn], err, 1))) break;
                        uint8_t *to = ring + (size_t)(turn * a.stages + st) * a.stage_bytes;
                        uint64_t *bar = &full[turn][st];
                        mbar_expect_tx(bar, (uint32_t)a.stage_tx);
#pragma unroll
                        for (int h = 0; h < HALVES; h++) {
                            uint8_t *half = to + h * a.chunks * (HALF_ROWS * 128);
                            if (a.whole_rows) tma_load_4d(half, &maps.codes[h], 0, it.tile * HALF_ROWS, p * (a.piece / 2), it.e, bar);
                            else
                                for (int c = 0; c < a.chunks; c++)
                                    tma_load_3d(half + c * (HALF_ROWS * 128), &maps.codes[h], p * (a.piece * 64) + c * 128, it.tile * HALF_ROWS, it.e, bar);
                            tma_load_3d(to + a.chunks * (2048 * U) + h * (HALF_ROWS * 2) * a.scale_pitch, &maps.scales[h], p * a.scale_cols, it.tile * HALF_ROWS, it.e, bar);
                        }
                        issued[turn]++;
                        if (++st == a.stages) { st = 0; parity[turn] ^= 1; }
                    }
                    turn ^= 1;
                }
                if (++tile == a.tiles && i + 1 < i1) { tile = 0; it = few_item<MODE>(a, here, ++slot, 0); }
                it.tile = tile;
            }
            // copies in flight must land before shared memory goes away
            for (int k = 0; k < 2; k++)
                for (int j = issued[k] - 1; j >= 0 && j >= issued[k] - a.stages; j--) mbar_wait(&full[k][j % a.stages], (uint32_t)(j / a.stages) & 1, err, 2);
        }
        return;
    }
    // ------------------------------------------------------------------------ products ----
    const int team = warp >> 3, gw = warp & 7, g = lane >> 2, t = lane & 3, gt = threadIdx.x & 255;
    const int wlog = a.w.group == 64 ? 1 : 0;
    pdl_wait();
    int slot = (int)(i0 / a.tiles), tile = (int)(i0 - (long long)slot * a.tiles), uses = 0, s = 0, ph = 0;      // s, ph: the team's stage, and the parity of its uses
    bool fresh = true;
    int have = -1;                                        // picks, gate/up: the row of x whose digits are there
    FewItem it{};
    // Lane row g is weight row wr: the two rows of a quarter of a warp are four apart, so that their pieces lie in different banks.
    const int wr = (g >> 1) | ((g & 1) << 2);
    int off[4];                                           // of this lane's pieces (words) in a chunk
#pragma unroll
    for (int j = 0; j < 4; j++) off[j] = WHOLE ? (((gw & 1) * 4 + t) ^ wr) * 16 : (((gw & 1) * 4 + j) ^ wr) * 16 + 4 * t;
    const int gx = min(g, NS - 1);                        // (lanes of columns behind the last read the last one's: what comes of it is not used)
#pragma unroll 1
    for (long long i = i0; i < i1; i++) {
        if (fresh) {
            it = few_item<MODE>(a, here, slot, tile);
            const int src = MODE == W4_GATEUP && a.idx ? it.first / a.topk : -1;      // (a token's picks: the same row)
            if (it.count && (src < 0 || src != have)) {
                have = src;
                few_digits<MODE, WHOLE, NS, IN>(a, it, blocks);
            }
            fresh = false;
        }
        it.tile = tile;
        if (it.count) {
            if (turn == team) {
                float acc[U][4] = {};
#pragma unroll 1
                for (int p = 0; p < pieces; p++) {
                    const uint8_t *st = ring + (size_t)(team * a.stages + s) * a.stage_bytes;
                    if (!(ok = ok && mbar_wait_all(&full[team][s], (uint32_t)ph, err, 3))) break;      // (the barriers below are met all the same)
                    const int nb = min(a.piece, a.blocks - p * a.piece);
                    // This warp's blocks are gw, gw + 8, ...: half a chunk of 128 bytes each, chunks HALF_ROWS * 128 apart, a row's 16-byte
                    // pieces at piece ^ (row & 7). Whatever does not change from block to block is taken out of the loop.
                    const uint8_t *cg = st + (gw >> 1) * (HALF_ROWS * 128) + wr * 128, *ch = cg + (MODE == W4_GATEUP ? a.chunks * 1024 : 1024);
                    const uint16_t *sg = reinterpret_cast<const uint16_t *>(st + a.chunks * (2048 * U)) + wr * a.scale_pitch + (WHOLE ? gw : (4 * gw) >> wlog), *sh = sg + 8 * a.scale_pitch;
                    const Block *bp = blocks + p * a.piece + gw;
                    const int first_group = (4 * (p * a.piece + gw)) >> wlog;
                    auto block = [&](int i, int sixteen, float (&acc)[4]) {
                        const uint8_t *pg = cg + i * (4 * HALF_ROWS * 128) + sixteen * 2048, *ph_ = ch + i * (4 * HALF_ROWS * 128) + sixteen * 2048;
                        const uint16_t *s_g = sg + sixteen * 16 * a.scale_pitch, *s_h = sh + sixteen * 16 * a.scale_pitch;
                        const Block &x = bp[8 * i];
                        uint4 vg, vh;
                        if (WHOLE) {
                            vg = *reinterpret_cast<const uint4 *>(pg + off[0]);
                            vh = *reinterpret_cast<const uint4 *>(ph_ + off[0]);
                        } else {
                            vg = make_uint4(*reinterpret_cast<const uint32_t *>(pg + off[0]), *reinterpret_cast<const uint32_t *>(pg + off[1]),
                                            *reinterpret_cast<const uint32_t *>(pg + off[2]), *reinterpret_cast<const uint32_t *>(pg + off[3]));
                            vh = make_uint4(*reinterpret_cast<const uint32_t *>(ph_ + off[0]), *reinterpret_cast<const uint32_t *>(ph_ + off[1]),
                                            *reinterpret_cast<const uint32_t *>(ph_ + off[2]), *reinterpret_cast<const uint32_t *>(ph_ + off[3]));
                        }
                        constexpr uint32_t LOW = 0x0f0f0f0fu;
                        // the block's scales (of four, two or one group) of rows g and g + 8
                        float fg[4], fh[4];
                        if (WHOLE) {
                            fg[0] = bf16_to_f32(s_g[8 * i]); fh[0] = bf16_to_f32(s_h[8 * i]);
                        } else if (wlog) {
                            const uint32_t g2 = *reinterpret_cast<const uint32_t *>(s_g + 16 * i), h2 = *reinterpret_cast<const uint32_t *>(s_h + 16 * i);
                            bf16x2_to_f32(g2, fg[0], fg[1]); bf16x2_to_f32(h2, fh[0], fh[1]);
                        } else {
                            const uint2 g4 = *reinterpret_cast<const uint2 *>(s_g + 32 * i), h4 = *reinterpret_cast<const uint2 *>(s_h + 32 * i);
                            bf16x2_to_f32(g4.x, fg[0], fg[1]); bf16x2_to_f32(g4.y, fg[2], fg[3]);
                            bf16x2_to_f32(h4.x, fh[0], fh[1]); bf16x2_to_f32(h4.y, fh[2], fh[3]);
                        }
                        if (!WHOLE) {
                            // a group behind the last (in a row's last block): zero, whatever lies there
                            const int left = a.w.groups - first_group - ((32 * i) >> wlog);
                            if (left < (4 >> wlog)) {
#pragma unroll
                                for (int k = 0; k < 4; k++) if (k >= left) { fg[k] = 0.f; fh[k] = 0.f; }
                            }
                        }
                        const uint4 x0 = x.digits[0][gx][t], x1 = x.digits[1][gx][t];
                        const float2 worth = *reinterpret_cast<const float2 *>(&x.worth[2 * t]);
                        float sum[4];
                        if (WHOLE) {
                            const int2 start = *reinterpret_cast<const int2 *>(&x.start[0][2 * t]);
                            int lo[4], hi[4];
                            few_mma(lo, vg.x & LOW, vh.x & LOW, vg.y & LOW, vh.y & LOW, x0.x, x0.y, 0, 0, 0, 0);
                            few_mma(hi, vg.x, vh.x, vg.y, vh.y, x1.x, x1.y, start.x, start.y, start.x, start.y);
                            few_mma(lo, vg.z & LOW, vh.z & LOW, vg.w & LOW, vh.w & LOW, x0.z, x0.w);
                            few_mma(hi, vg.z, vh.z, vg.w, vh.w, x1.z, x1.w);
#pragma unroll
                            for (int q = 0; q < 4; q++) sum[q] = few_float<true>(hi[q] + 16 * lo[q]) * (q < 2 ? fg[0] : fh[0]);
                        } else {
                            int c[4];
#pragma unroll
                            for (int q = 0; q < 4; q++) sum[q] = 0.f;
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const uint32_t rg = word_of(vg, j), rh = word_of(vh, j);
                                if (wlog == 0 || !(j & 1)) {
                                    const int2 start = *reinterpret_cast<const int2 *>(&x.start[WHOLE ? 0 : j][2 * t]);
                                    c[0] = start.x; c[1] = start.y; c[2] = start.x; c[3] = start.y;
                                }
                                const uint4 &d = j < 2 ? x0 : x1;
                                few_mma(c, rg & LOW, rh & LOW, (rg >> 4) & LOW, (rh >> 4) & LOW, j & 1 ? d.z : d.x, j & 1 ? d.w : d.y);
                                if (wlog == 0 || (j & 1)) {
                                    const float sg_ = wlog ? fg[j >> 1] : fg[j], sh_ = wlog ? fh[j >> 1] : fh[j];
#pragma unroll
                                    for (int q = 0; q < 4; q++) sum[q] = fmaf(few_float<false>(c[q]), q < 2 ? sg_ : sh_, sum[q]);
                                }
                            }
                        }
                        // (a digit's worth comes last: times a scale alone it may be too small or too large for FP32)
#pragma unroll
                        for (int q = 0; q < 4; q++) acc[q] = fmaf(sum[q], q & 1 ? worth.y : worth.x, acc[q]);
                    };
constexpr int MOST = FW_PIECE / 1024 / U;
                    if (nb == 8 * MOST) {                // (no branch keeps the blocks apart)
#pragma unroll
                        for (int i = 0; i < MOST; i++)
#pragma unroll
                            for (int k = 0; k < U; k++) block(i, k, acc[k]);
                    } else
#pragma unroll 1
                        for (int i = 0; i < MOST; i++) {
                            if (gw + 8 * i >= nb) break;
#pragma unroll
                            for (int k = 0; k < U; k++) block(i, k, acc[k]);
                        }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&empty[team][s]);
                    if (++s == a.stages) { s = 0; ph ^= 1; }
                }
                float (*sum)[16 * U][FW_COLS] = s_sum[team][uses & 1];
                uses++;
#pragma unroll
                for (int k = 0; k < U; k++) {
                    *reinterpret_cast<float2 *>(&sum[gw][16 * k + wr][2 * t]) = make_float2(acc[k][0], acc[k][1]);
                    *reinterpret_cast<float2 *>(&sum[gw][16 * k + wr + 8][2 * t]) = make_float2(acc[k][2], acc[k][3]);
                }
                bar_sync(2 + team, 256);
                constexpr int OUT = MODE == W4_GATEUP ? 8 : 16 * U;           // outputs of a row of x
                if (gt < OUT * it.count) {
                    const int r = gt & (OUT - 1), k = gt / OUT, col = k * FW_DIGITS;
                    auto total = [&](int r) {            // digit by digit, the least first
                        float4 d = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int w = 0; w < 8; w++) {
                            const float4 in = *reinterpret_cast<const float4 *>(&sum[w][r][col]);
                            d.x += in.x; d.y += in.y; d.z += in.z; d.w += in.w;
                        }
                        return (((d.x + d.y) + d.z) + d.w) * FW_REST;
                    };
                    float v = total(r);
                    const float u = MODE == W4_GATEUP ? total(r + 8) : 0.f;
                    if (MODE == W4_GATEUP) v = swiglu_value(v, u, a.limit);
                    const int row = it.tile * OUT + r;
                    const size_t at = (size_t)(it.first + k) * a.ldy + row;
                    if (row < a.w.rows) {
                        if (a.y_dt == DT_F32) static_cast<float *>(a.y)[at] = v;
                        else static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(v);
                    }
                }
            }
            turn ^= 1;
        }
        if (++tile == a.tiles) { tile = 0; slot++; fresh = true; }
    }
}

template <typename IN, int MODE, bool WHOLE, int NS, int U>
static int few_launch(cudaStream_t st, const FewMaps &m, FewArgs &a, bool early)
{
    static SmemGrant grant;
    const int digit_bytes = (int)sizeof(FewBlock<NS, WHOLE>) * a.blocks;
    a.stages = std::min((FW_SMEM - (U - 1) * FW_SUMS - digit_bytes) / a.stage_bytes / 2, FW_MAX_STAGES);
    const size_t smem = 1024 + (size_t)2 * a.stages * a.stage_bytes + digit_bytes;
    if (a.stages < 1) { set_last_error("a 4-bit product has no room for its stages"); return -1; }
    // (what counts is this and the sums: more than 48 KB of them must be asked for)
    if (!dev_opt_in_smem((const void *)w4_few_kernel<IN, MODE, WHOLE, NS, U>, std::max(smem, (size_t)64 * 1024), grant)) return -1;
    const long long items = (long long)a.tiles * (MODE == W4_DENSE ? 1 : a.idx ? a.n : a.slots.max);
    const int grid = (int)std::min<long long>(items, dev_sms());
    if (early) G5B_LAUNCH_PDL((w4_few_kernel<IN, MODE, WHOLE, NS, U>), dim3(grid), dim3(FW_THREADS), smem, st, m, a);
    else       G5B_LAUNCH((w4_few_kernel<IN, MODE, WHOLE, NS, U>), grid, FW_THREADS, smem, st, m, a);
    return 0;
}
template <typename IN, int MODE, bool WHOLE>
static int few_columns(cudaStream_t st, const FewMaps &m, FewArgs &a, bool early)
{
    if constexpr (MODE != W4_GATEUP)
        if (a.sixteens == 2)
            return a.per == 1 ? few_launch<IN, MODE, WHOLE, FW_DIGITS, 2>(st, m, a, early) : few_launch<IN, MODE, WHOLE, FW_COLS, 2>(st, m, a, early);
    return a.per == 1 ? few_launch<IN, MODE, WHOLE, FW_DIGITS, 1>(st, m, a, early) : few_launch<IN, MODE, WHOLE, FW_COLS, 1>(st, m, a, early);
}
template <typename IN, int MODE>
static int few_group(cudaStream_t st, const FewMaps &m, FewArgs &a, bool early)
{
    return a.w.group == 128 ? few_columns<IN, MODE, true>(st, m, a, early) : few_columns<IN, MODE, false>(st, m, a, early);
}

// What a block's digits take: of one row, of two.
static size_t few_block(int rows) { return rows > 1 ? sizeof(FewBlock<FW_COLS, false>) : sizeof(FewBlock<FW_DIGITS, false>); }
// Rows of a tile for a matrix of so many columns: two if there is room for their digits, else one or none.
int w4_few_rows(int cols)
{
    const size_t blocks = w4_kp(cols) / 128;
    return blocks * few_block(FW_ROWS) <= (size_t)FW_DIGIT_BYTES ? FW_ROWS : blocks * few_block(1) <= (size_t)FW_DIGIT_BYTES ? 1 : 0;
}

int w4_few(cudaStream_t st, const W4Job &j)
{
    FewArgs a{};
    const int size = j.x_dt == DT_F32 ? 4 : 2;
    a.w = j.w; a.x = j.x; a.ldx = j.ldx; a.x_dt = j.x_dt; a.cols = j.w.cols; a.blocks = w4_kp(j.w.cols) / 128;
    a.wide = reinterpret_cast<uintptr_t>(j.x) % 16 == 0 && j.ldx * size % 16 == 0;
    a.rows = j.T; a.per = j.mode == W4_DENSE ? j.T : j.idx ? 1 : j.slots.rows; a.order = j.order; a.idx = j.idx; a.topk = j.topk; a.E = j.count; a.n = j.T; a.slots = j.slots;
    a.y = j.y; a.ldy = j.ldy; a.y_dt = j.y_dt; a.limit = j.limit;
    const int slots = j.mode == W4_DENSE ? 1 : j.idx ? j.T : j.slots.max;
    // (two sixteens to an item wherever it has two blocks of 128 columns to a warp at most, and a CTA still has two such items)
    a.sixteens = j.mode != W4_GATEUP && a.blocks <= FW_PIECE / 256 && (long long)slots * j.w.rows >= 64ll * dev_sms() ? 2 : 1;
    const int half_rows = j.mode == W4_GATEUP ? 8 : 16 * a.sixteens;
    a.tiles = (j.w.rows + half_rows - 1) / half_rows;
    a.whole_rows = j.w.pitch % 128 == 0;
    // Two stages of each team at least: with many digits beside them in pieces of half the columns.
    const size_t digits = (size_t)a.blocks * few_block(a.per);
    for (a.piece = FW_PIECE / 128;; a.piece /= 2) {
        a.chunks = std::min(a.piece / 2, (j.w.pitch + 127) / 128);
        a.scale_cols = std::min(a.piece * 128 / j.w.group, j.w.sp);
        a.scale_pitch = a.scale_cols + 8;
        a.stage_tx = (a.chunks * 2048 + 32 * a.scale_pitch) * a.sixteens;
        a.stage_bytes = (a.stage_tx + 1023) / 1024 * 1024;
        if (a.piece < FW_PIECE / 128 || 4 * (size_t)a.stage_bytes + (a.sixteens - 1) * FW_SUMS + digits <= (size_t)FW_SMEM) break;
    }
    FewMaps m;
    for (int h = 0; h < 2; h++) {
        const W4Mat &w = h && j.mode == W4_GATEUP ? j.up : j.w;
        if (h && j.mode != W4_GATEUP) { m.codes[1] = m.codes[0]; m.scales[1] = m.scales[0]; break; }
        const cuuint64_t pitch = (cuuint64_t)w.pitch, rows = (cuuint64_t)w.rows, count = (cuuint64_t)j.count;
        const cuuint64_t size4[4] = {128, rows, pitch / 128, count}, stride4[3] = {pitch, 128, (cuuint64_t)w.codes_stride}, size3[3] = {pitch, rows, count}, stride3[2] = {pitch, (cuuint64_t)w.codes_stride};
        const cuuint32_t box4[4] = {128, (cuuint32_t)half_rows, (cuuint32_t)a.chunks, 1}, box3[3] = {128, (cuuint32_t)half_rows, 1};
        const cuuint64_t ssize[3] = {(cuuint64_t)w.sp, rows, count}, sstride[2] = {(cuuint64_t)w.sp * 2, (cuuint64_t)w.scales_stride * 2};
        const cuuint32_t sbox[3] = {(cuuint32_t)a.scale_pitch, (cuuint32_t)half_rows, 1};
        const bool codes = a.whole_rows ? tc_encode_swizzled(&m.codes[h], w.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, size4, stride4, box4, CU_TENSOR_MAP_SWIZZLE_128B)
                                        : tc_encode_swizzled(&m.codes[h], w.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, size3, stride3, box3, CU_TENSOR_MAP_SWIZZLE_128B);
        if (!codes || !tc_encode_swizzled(&m.scales[h], w.scales, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, ssize, sstride, sbox, CU_TENSOR_MAP_SWIZZLE_NONE)) {
            set_last_error("a tensor map of a 4-bit product was refused");
            return -1;
        }
    }
    if (j.mode == W4_DOWN) return few_group<float, W4_DOWN>(st, m, a, j.early);
    if (j.x_dt == DT_BF16) return j.mode == W4_DENSE ? few_group<uint16_t, W4_DENSE>(st, m, a, j.early) : few_group<uint16_t, W4_GATEUP>(st, m, a, j.early);
    return j.mode == W4_DENSE ? few_group<float, W4_DENSE>(st, m, a, j.early) : few_group<float, W4_GATEUP>(st, m, a, j.early);
}

int w4_few_status(cudaStream_t st) { return w4_flag(g_few_err, st); }

}  // namespace g5b
