// w4_few.cu - 4-bit weights times at most eight columns of activations (terms of rows): one decoded token, a few sequences, the few
// tokens of an expert in a batch.
//
// Bound by HBM: half a byte and a scale's share per weight. The legacy matrix instruction does the products (16 weight rows x 16
// columns x 8 activation columns); the 5th-generation tensor cores would need 128 rows at a time and hand-overs of their sums.
// One CTA per SM, persistent. Work comes in items of 16 weight rows (gate/up: eight gate rows and the eight up rows that go with them),
// in pieces of 4096 columns; a CTA takes a contiguous share of them.
//   warp 16   brings an item's rows into a ring in shared memory, one TMA load for the codes and one for the scales (gate/up: two
//             each), as many ahead as fit: they wait for nothing but room, so HBM is busy while sums are put together and rows change.
//             (A bulk copy per row was 125 cycles of issue each: 2.3 TB/s.)
//   0-7, 8-15 take items in turn; the eight warps of a team share an item's blocks of 128 columns, and their sums meet in shared
//             memory in a fixed order
//   codes     a lane takes 16 bytes of rows g and g + 8 (lane = 4 g + t), a quad 64 bytes: 128 columns of each. Nibbles become F16
//             pairs without a conversion: (code | 0x6400) is 1024 + code, (16 code | 0x6400) is 1024 + 16 code, and one packed operation
//             takes the offset (and the 16) off, exactly. A pair is columns i and i + 4 of a word's eight; which column stands for
//             which k of an MMA does not matter as long as both operands agree, and the activations lie in that order.
//   scales    in FP32, once per group, on the sums of the group. A quad's 128 columns are one group of 128; for smaller groups
//             a lane takes its words 16 bytes apart, so that every pair of MMAs is 32 columns of one group.
//   x         becomes F16 terms in shared memory whenever the rows change (dense: once; experts: with the expert), in the order in
//             which the lanes read them: F32 rows two terms (22 significant bits of the row's largest), BF16 rows one, exact.
// Sums are FP32: in the tensor cores over a group, outside across groups.
// Every wait is bounded: one that runs out sets a flag (g5b_w4_status).
#include <algorithm>

#include "tc_ptx.cuh"
#include "w4.cuh"

namespace g5b {

constexpr int FW_WARPS = 16, FW_THREADS = (FW_WARPS + 1) * 32;
constexpr int FW_COLS = 8;                           // activation columns
constexpr int FW_PIECE = 4096;                       // weight columns of a stage: 16 chunks of 256 (128 bytes)
constexpr int FW_TERM_BYTES = 64 * 1024;             // room for the terms
constexpr int FW_MAX_STAGES = 12;
constexpr int FW_SMEM = 206 * 1024;                  // for stages and terms (17 KB of sums beside them)

static __device__ int g_few_err;                     // a wait that ran out: its code (0: none)

struct FewMaps { CUtensorMap codes[2], scales[2]; };  // gate/up: of either; else the first
struct FewArgs {
    W4Mat w;
    const void *x;
    size_t ldx;
    int x_dt, cols, blocks;        // columns of x, blocks of 128 of them
    int wide;                      // x may be read 16 bytes at a time
    int tiles, rows;               // row tiles; dense: rows of x
    const int *order, *idx;        // experts: sorted picks, or (idx) the picks themselves, each a slot of its own
    int topk, E, n;
    W4Slots slots;
    void *y;
    size_t ldy;
    int y_dt;
    float limit;
    int whole_rows;                // rows of codes are whole chunks: one load brings all of a stage's
    int chunks, scale_cols;        // of a stage at most
    int scale_pitch;               // scales of a stage's row: eight more, so that eight rows lie in different banks
    int stages, stage_bytes, stage_tx;
};
struct FewItem { int e, first, count, tile; };       // expert; sorted rows (dense: rows of x); row tile
template <int MODE>
__device__ __forceinline__ int few_slots(const FewArgs &a) { return MODE == W4_DENSE ? 1 : a.idx ? a.n : __ldg(a.slots.n); }
template <int MODE>
__device__ __forceinline__ FewItem few_item(const FewArgs &a, int slot, int tile)
{
    if (MODE == W4_DENSE) return FewItem{0, 0, a.rows, tile};
    if (a.idx) {
        const int e = __ldg(a.idx + slot);
        return FewItem{e, slot, e >= 0 && e < a.E ? 1 : 0, tile};
    }
    return FewItem{__ldg(a.slots.expert + slot), __ldg(a.slots.first + slot), __ldg(a.slots.count + slot), tile};
}

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
// (not volatile: two blocks' chains of these are put side by side)
__device__ __forceinline__ void few_mma(float (&c)[4], const uint32_t (&g)[4], const uint32_t (&h)[4], int k, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(g[k]), "r"(h[k]), "r"(g[k + 1]), "r"(h[k + 1]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t word_of(const uint4 &v, int j) { return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w; }

__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// Eight values from column c on, zero behind the last.
template <typename IN>
__device__ __forceinline__ void few_load8(float (&v)[8], const IN *row, int c, int cols, bool wide);
template <>
__device__ __forceinline__ void few_load8<float>(float (&v)[8], const float *row, int c, int cols, bool wide)
{
    if (wide && c + 8 <= cols) {
        const float4 a = *reinterpret_cast<const float4 *>(row + c), b = *reinterpret_cast<const float4 *>(row + c + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = c + i < cols ? row[c + i] : 0.f;
}
template <>
__device__ __forceinline__ void few_load8<uint16_t>(float (&v)[8], const uint16_t *row, int c, int cols, bool wide)
{
    if (wide && c + 8 <= cols) {
        const uint4 a = *reinterpret_cast<const uint4 *>(row + c);
        bf16x2_to_f32(a.x, v[0], v[1]); bf16x2_to_f32(a.y, v[2], v[3]); bf16x2_to_f32(a.z, v[4], v[5]); bf16x2_to_f32(a.w, v[6], v[7]);
    } else
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = c + i < cols ? bf16_to_f32(row[c + i]) : 0.f;
}

// The 512 consumer threads: rows of an item as terms. terms: [block][j][column][t] 16 bytes, as the lanes read them; inv: 2^-e of each row.
// The power of two brings the row's largest magnitude below 2^14; what falls below F16's 2^-24 then is 2^-38 of it.
template <int TERMS, int MODE, bool WHOLE, int NS, typename IN>
__device__ __forceinline__ void few_terms(const FewArgs &a, const FewItem &it, uint4 *terms, float *inv, uint32_t *s_max)
{
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = it.count <= 1 ? 1 : it.count <= 2 ? 2 : it.count <= 4 ? 4 : 8, per = FW_WARPS / rows;    // warps to a row
    const int i = warp / per, c_first = ((warp - i * per) * 32 + lane) * 8, c_step = per * 256;
    const bool live = i < it.count;
    const int at = it.first + (live ? i : 0);
    const int src = MODE != W4_GATEUP ? at : (a.idx ? at : __ldg(a.order + at)) / a.topk;
    const IN *row = static_cast<const IN *>(a.x) + (size_t)src * a.ldx;
    uint32_t m = 0;
    if (live)
        for (int c = c_first; c < a.cols; c += c_step) {
            float v[8];
            few_load8<IN>(v, row, c, a.cols, a.wide);
#pragma unroll
            for (int k = 0; k < 8; k++) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
        }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) s_max[warp] = m;
    bar_sync(1, FW_WARPS * 32);                          // (and nobody reads the terms of the rows before any more)
    for (int k = 0; k < per; k++) m = max(m, s_max[i * per + k]);
    const bool finite = m < 0x7f800000u;
    // 2^(e - 1) <= max < 2^e (a subnormal one counts as 2^-126)
    const int e = max((int)(m >> 23), 1) - 126, up = min(14 - e, 126);
    const float scale = __int_as_float((up + 127) << 23);
    if (live && (threadIdx.x & (per * 32 - 1)) == 0) inv[i] = finite ? __int_as_float((127 - up) << 23) : __int_as_float(0x7fc00000);
    if (live)
        for (int c = c_first; c < a.blocks * 128; c += c_step) {
            float v[8];
            few_load8<IN>(v, row, c, a.cols, a.wide);
            __align__(16) __half h[8], l[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int to = (k & 3) * 2 + (k >> 2);                  // 0 4 1 5 2 6 3 7
                const float f = finite ? v[k] * scale : 0.f;
                h[to] = __float2half_rn(f);
                l[to] = __float2half_rn(f - __half2float(h[to]));
            }
            const int w = (c & 127) >> 3, j = WHOLE ? w & 3 : w >> 2, t = WHOLE ? w >> 2 : w & 3;
            uint4 *to = terms + (((c >> 7) * 4 + j) * NS + i * TERMS) * 4 + t;
            to[0] = *reinterpret_cast<const uint4 *>(h);
            if (TERMS == 2) to[4] = *reinterpret_cast<const uint4 *>(l);
        }
    bar_sync(1, FW_WARPS * 32);
}

// WHOLE: groups of 128. NS: columns that the terms have room for.
template <int TERMS, int MODE, bool WHOLE, int NS>
__global__ void __launch_bounds__(FW_THREADS, 1) w4_few_kernel(const __grid_constant__ FewMaps maps, const FewArgs a)
{
    constexpr int HALVES = MODE == W4_GATEUP ? 2 : 1, HALF_ROWS = 16 / HALVES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    uint8_t *ring = smem;                                                             // [stages][half][chunk][row][128] codes, [half][row][scale_cols] scales
    uint4 *terms = reinterpret_cast<uint4 *>(smem + (size_t)a.stages * a.stage_bytes);
    __shared__ uint64_t full[FW_MAX_STAGES], empty[FW_MAX_STAGES];
    __shared__ float s_sum[2][2][8][16][FW_COLS];                                     // [team][item's parity][warp][row][column]
    __shared__ float s_inv[FW_COLS];
    __shared__ uint32_t s_max[FW_WARPS];
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    int *err = &g_few_err;
    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (MODE != W4_DENSE && !a.idx) pdl_wait();           // (the slots are another kernel's)
    const int pieces = (a.blocks + FW_PIECE / 128 - 1) / (FW_PIECE / 128);
    const long long items = (long long)few_slots<MODE>(a) * a.tiles;
    const long long i0 = items * blockIdx.x / gridDim.x, i1 = items * (blockIdx.x + 1) / gridDim.x;
    bool ok = true;
    int s = 0, ph = 0;                                    // stage, and the parity of its uses

    if (warp == FW_WARPS) {
        // ------------------------------------------------------------------- weights ----
        if (elect_one()) {
            int slot = (int)(i0 / a.tiles), tile = (int)(i0 - (long long)slot * a.tiles), issued = 0;
            FewItem it = i0 < i1 ? few_item<MODE>(a, slot, tile) : FewItem{};
#pragma unroll 1
            for (long long i = i0; i < i1 && ok; i++) {
                if (it.count) {
#pragma unroll 1
                    for (int p = 0; p < pieces; p++) {
                        if (issued >= a.stages && !(ok = mbar_wait(&empty[s], (uint32_t)(ph ^ 1), err, 1))) break;
                        uint8_t *to = ring + (size_t)s * a.stage_bytes;
                        mbar_expect_tx(&full[s], (uint32_t)a.stage_tx);
#pragma unroll
                        for (int h = 0; h < HALVES; h++) {
                            uint8_t *half = to + h * a.chunks * (HALF_ROWS * 128);
                            if (a.whole_rows) tma_load_4d(half, &maps.codes[h], 0, it.tile * HALF_ROWS, p * 16, it.e, &full[s]);
                            else
                                for (int c = 0; c < a.chunks; c++)
                                    tma_load_3d(half + c * (HALF_ROWS * 128), &maps.codes[h], p * (FW_PIECE / 2) + c * 128, it.tile * HALF_ROWS, it.e, &full[s]);
                            tma_load_3d(to + a.chunks * 2048 + h * (HALF_ROWS * 2) * a.scale_pitch, &maps.scales[h], p * a.scale_cols, it.tile * HALF_ROWS, it.e, &full[s]);
                        }
                        issued++;
                        if (++s == a.stages) { s = 0; ph ^= 1; }
                    }
                }
                if (++tile == a.tiles && i + 1 < i1) { tile = 0; it = few_item<MODE>(a, ++slot, 0); }
                it.tile = tile;
            }
            // copies in flight must land before shared memory goes away
            for (int j = issued - 1; j >= 0 && j >= issued - a.stages; j--) mbar_wait(&full[j % a.stages], (uint32_t)(j / a.stages) & 1, err, 2);
        }
        return;
    }
    // ------------------------------------------------------------------------ products ----
    const int team = warp >> 3, gw = warp & 7, g = lane >> 2, t = lane & 3, gt = threadIdx.x & 255;
    const int wlog = a.w.group == 64 ? 1 : 0;
    pdl_wait();
    int slot = (int)(i0 / a.tiles), tile = (int)(i0 - (long long)slot * a.tiles), turn = 0, uses = 0;
    bool fresh = true;
    FewItem it{};
    // Lane row g is weight row wr: the two rows of a quarter of a warp are four apart, so that their pieces lie in different banks.
    const int wr = (g >> 1) | ((g & 1) << 2);
    int off[4];                                           // of this lane's pieces (words) in a chunk
#pragma unroll
    for (int j = 0; j < 4; j++) off[j] = WHOLE ? (((gw & 1) * 4 + t) ^ wr) * 16 : (((gw & 1) * 4 + j) ^ wr) * 16 + 4 * t;
    // (lanes of columns behind the last read the last one's: what comes of it is not used)
    const uint4 *xt = terms + min(g, NS - 1) * 4 + t;
#pragma unroll 1
    for (long long i = i0; i < i1; i++) {
        if (fresh) {
            it = few_item<MODE>(a, slot, tile);
            if (it.count) {
                if (MODE == W4_DOWN || a.x_dt == DT_F32) few_terms<TERMS, MODE, WHOLE, NS, float>(a, it, terms, s_inv, s_max);
                else                                     few_terms<TERMS, MODE, WHOLE, NS, uint16_t>(a, it, terms, s_inv, s_max);
            }
            fresh = false;
        }
        it.tile = tile;
        if (it.count) {
            if (turn == team) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                for (int p = 0; p < pieces; p++) {
                    const uint8_t *st = ring + (size_t)s * a.stage_bytes;
                    if (!(ok = ok && mbar_wait_all(&full[s], (uint32_t)ph, err, 3))) break;      // (the barriers below are met all the same)
                    const int nb = min(FW_PIECE / 128, a.blocks - p * (FW_PIECE / 128));
                    // This warp's blocks are gw, gw + 8, ...: half a chunk of 128 bytes each, chunks HALF_ROWS * 128 apart, a row's 16-byte
                    // pieces at piece ^ (row & 7). Whatever does not change from block to block is taken out of the loop.
                    const uint8_t *cg = st + (gw >> 1) * (HALF_ROWS * 128) + wr * 128, *ch = cg + (MODE == W4_GATEUP ? a.chunks * 1024 : 1024);
                    const uint16_t *sg = reinterpret_cast<const uint16_t *>(st + a.chunks * 2048) + wr * a.scale_pitch + (WHOLE ? gw : (4 * gw) >> wlog), *sh = sg + 8 * a.scale_pitch;
                    const uint4 *xp = xt + (p * (FW_PIECE / 128) + gw) * (4 * NS * 4);
                    const int first_group = (4 * (p * (FW_PIECE / 128) + gw)) >> wlog;
                    // two blocks at a time (the second may not be there): their chains of eight dependent products side by side
                    auto pair = [&](int i, bool both) {
                        uint4 vg[2], vh[2];
                        float c[2][4];
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            if (u && !both) break;
                            const uint8_t *pg = cg + (i + u) * (4 * HALF_ROWS * 128), *ph_ = ch + (i + u) * (4 * HALF_ROWS * 128);
                            if (WHOLE) {
                                vg[u] = *reinterpret_cast<const uint4 *>(pg + off[0]);
                                vh[u] = *reinterpret_cast<const uint4 *>(ph_ + off[0]);
                            } else {
                                vg[u] = make_uint4(*reinterpret_cast<const uint32_t *>(pg + off[0]), *reinterpret_cast<const uint32_t *>(pg + off[1]),
                                                   *reinterpret_cast<const uint32_t *>(pg + off[2]), *reinterpret_cast<const uint32_t *>(pg + off[3]));
                                vh[u] = make_uint4(*reinterpret_cast<const uint32_t *>(ph_ + off[0]), *reinterpret_cast<const uint32_t *>(ph_ + off[1]),
                                                   *reinterpret_cast<const uint32_t *>(ph_ + off[2]), *reinterpret_cast<const uint32_t *>(ph_ + off[3]));
                            }
#pragma unroll
                            for (int q = 0; q < 4; q++) c[u][q] = 0.f;
                        }
#pragma unroll
                        for (int j = 0; j < 4; j++)
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                if (u && !both) break;
                                const uint4 x = xp[((i + u) * 8 * 4 + j) * (NS * 4)];
                                uint32_t wg[4], wh[4];
                                const uint32_t rg = word_of(vg[u], j), rh = word_of(vh[u], j);
                                nibbles(rg, wg[0], wg[1]); nibbles(rg >> 8, wg[2], wg[3]);
                                nibbles(rh, wh[0], wh[1]); nibbles(rh >> 8, wh[2], wh[3]);
                                few_mma(c[u], wg, wh, 0, x.x, x.y);
                                few_mma(c[u], wg, wh, 2, x.z, x.w);
                                if (!WHOLE || j == 3) {
                                    // (groups smaller than a block: one behind the last is zero, whatever lies there)
                                    const int k = WHOLE ? 8 * (i + u) : (32 * (i + u) + j) >> wlog;
                                    const bool here = WHOLE || first_group + k < a.w.groups;
                                    const float fg = here ? bf16_to_f32(sg[k]) : 0.f, fh = here ? bf16_to_f32(sh[k]) : 0.f;
                                    acc[0] = fmaf(c[u][0], fg, acc[0]); acc[1] = fmaf(c[u][1], fg, acc[1]);
                                    acc[2] = fmaf(c[u][2], fh, acc[2]); acc[3] = fmaf(c[u][3], fh, acc[3]);
#pragma unroll
                                    for (int q = 0; q < 4; q++) c[u][q] = 0.f;
                                }
                            }
                    };
#pragma unroll
                    for (int i = 0; i < FW_PIECE / 1024; i += 2) {
                        if (gw + 8 * (i + 1) < nb) pair(i, true);
                        else if (gw + 8 * i < nb) pair(i, false);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&empty[s]);
                    if (++s == a.stages) { s = 0; ph ^= 1; }
                }
                float (*sum)[16][FW_COLS] = s_sum[team][uses & 1];
                uses++;
                *reinterpret_cast<float2 *>(&sum[gw][wr][2 * t]) = make_float2(acc[0], acc[1]);
                *reinterpret_cast<float2 *>(&sum[gw][wr + 8][2 * t]) = make_float2(acc[2], acc[3]);
                bar_sync(2 + team, 256);
                constexpr int OUT = MODE == W4_GATEUP ? 8 : 16;           // outputs of a row of x
                if (gt < OUT * it.count) {
                    const int r = gt & (OUT - 1), k = gt / OUT;
                    float v = 0.f, u = 0.f;
#pragma unroll
                    for (int w = 0; w < 8; w++)
#pragma unroll
                        for (int m = TERMS - 1; m >= 0; m--) {
                            v += sum[w][r][k * TERMS + m];
                            if (MODE == W4_GATEUP) u += sum[w][r + 8][k * TERMS + m];
                        }
                    const float inv = s_inv[k];
                    v *= inv;
                    if (MODE == W4_GATEUP) v = swiglu_value(v, u * inv, a.limit);
                    const int row = it.tile * OUT + r;
                    const size_t at = (size_t)(it.first + k) * a.ldy + row;
                    if (row < a.w.rows) {
                        if (a.y_dt == DT_F32) static_cast<float *>(a.y)[at] = v;
                        else static_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(v);
                    }
                }
            } else {
                // the other eight warps' item
                s += pieces;
                while (s >= a.stages) { s -= a.stages; ph ^= 1; }
            }
            turn ^= 1;
        }
        if (++tile == a.tiles) { tile = 0; slot++; fresh = true; }
    }
}

template <int TERMS, int MODE, bool WHOLE, int NS>
static int few_launch(cudaStream_t st, const FewMaps &m, FewArgs &a, bool early)
{
    static SmemGrant grant;
    const int term_bytes = NS * a.blocks * 256;
    a.stages = std::min((FW_SMEM - term_bytes) / a.stage_bytes, FW_MAX_STAGES);
    const size_t smem = 1024 + (size_t)a.stages * a.stage_bytes + term_bytes;
    if (a.stages < 2) { set_last_error("a 4-bit product has no room for its stages"); return -1; }
    // (what counts is this and the 17 KB of sums: more than 48 KB of them must be asked for)
    if (!dev_opt_in_smem((const void *)w4_few_kernel<TERMS, MODE, WHOLE, NS>, std::max(smem, (size_t)64 * 1024), grant)) return -1;
    const long long items = (long long)a.tiles * (MODE == W4_DENSE ? 1 : a.idx ? a.n : a.slots.max);
    const int grid = (int)std::min<long long>(items, dev_sms());
    if (early) G5B_LAUNCH_PDL((w4_few_kernel<TERMS, MODE, WHOLE, NS>), dim3(grid), dim3(FW_THREADS), smem, st, m, a);
    else       G5B_LAUNCH((w4_few_kernel<TERMS, MODE, WHOLE, NS>), grid, FW_THREADS, smem, st, m, a);
    return 0;
}
template <int TERMS, int MODE>
static int few_group(cudaStream_t st, const FewMaps &m, FewArgs &a, bool early)
{
    const bool one = MODE == W4_DENSE ? a.rows == 1 : a.idx != nullptr;              // a row at a time
    if (a.w.group == 128) return one ? few_launch<TERMS, MODE, true, TERMS>(st, m, a, early) : few_launch<TERMS, MODE, true, FW_COLS>(st, m, a, early);
    return one ? few_launch<TERMS, MODE, false, TERMS>(st, m, a, early) : few_launch<TERMS, MODE, false, FW_COLS>(st, m, a, early);
}

// Rows of a tile: eight columns of terms if there is room for them, else one row if there is for that.
int w4_few_rows(int n_terms, int cols)
{
    const int kp = w4_kp(cols);
    return 2 * kp * FW_COLS <= FW_TERM_BYTES ? FW_COLS / n_terms : 2 * kp * n_terms <= FW_TERM_BYTES ? 1 : 0;
}

int w4_few(cudaStream_t st, const W4Job &j)
{
    FewArgs a{};
    const int size = j.x_dt == DT_F32 ? 4 : 2;
    a.w = j.w; a.x = j.x; a.ldx = j.ldx; a.x_dt = j.x_dt; a.cols = j.w.cols; a.blocks = w4_kp(j.w.cols) / 128;
    a.wide = reinterpret_cast<uintptr_t>(j.x) % 16 == 0 && j.ldx * size % 16 == 0;
    a.tiles = (j.w.rows + (j.mode == W4_GATEUP ? 7 : 15)) / (j.mode == W4_GATEUP ? 8 : 16);
    a.rows = j.T; a.order = j.order; a.idx = j.idx; a.topk = j.topk; a.E = j.count; a.n = j.T; a.slots = j.slots;
    a.y = j.y; a.ldy = j.ldy; a.y_dt = j.y_dt; a.limit = j.limit;
    const int half_rows = j.mode == W4_GATEUP ? 8 : 16;
    a.whole_rows = j.w.pitch % 128 == 0;
    a.chunks = std::min(16, (j.w.pitch + 127) / 128);
    a.scale_cols = std::min(FW_PIECE / j.w.group, j.w.sp);
    a.scale_pitch = a.scale_cols + 8;
    a.stage_tx = a.chunks * 2048 + 32 * a.scale_pitch;
    a.stage_bytes = (a.stage_tx + 1023) / 1024 * 1024;
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
    if (j.n_terms == 1)
        return j.mode == W4_DENSE ? few_group<1, W4_DENSE>(st, m, a, j.early) : j.mode == W4_GATEUP ? few_group<1, W4_GATEUP>(st, m, a, j.early) : few_group<1, W4_DOWN>(st, m, a, j.early);
    return j.mode == W4_DENSE ? few_group<2, W4_DENSE>(st, m, a, j.early) : j.mode == W4_GATEUP ? few_group<2, W4_GATEUP>(st, m, a, j.early) : few_group<2, W4_DOWN>(st, m, a, j.early);
}

int w4_few_status(cudaStream_t st) { return w4_flag(g_few_err, st); }

}  // namespace g5b
