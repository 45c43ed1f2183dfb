// expert_rows.cu - tokens sorted by expert and back.
//
// sort     picks p = token * topk + k of experts in [0, E) in the order of (expert, p): order[i] = p, place[p] = i (-1 for a
//          pick of no expert here; order is -1 behind the last), offsets[e] = picks of the experts before e.
// gather   rows[i] = x[order[i] / topk]
// combine  out[t] = sum over k of w[t][k] rows[place[t][k]], in the order of k
//
// The sort counts, it compares nothing: a warp owns a stretch of the picks, counts its experts 32 picks at a time (lanes with
// the same expert find each other with one match instruction, so a warp's counts need no atomics and the order of equal
// experts is that of the picks), counts become first places by sums over warps, CTAs and experts, and a second pass over the
// stretch places the picks. One launch: a CTA alone up to SORT_ALONE picks, beyond a cluster of eight whose CTAs read each
// other's counts through distributed shared memory. Bound by the latency of those steps.
#include <type_traits>

#include "common.cuh"
#include "w4.h"

namespace g5b {

constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32, SORT_CLUSTER = 8;
constexpr int SORT_ALONE = 4096;
constexpr int SORT_HELD = SORT_ALONE / (SORT_WARPS * 32);      // picks of a lane that stay in registers

__device__ __forceinline__ int ld_cluster_s32(const int *p, uint32_t rank)
{
    uint32_t theirs;
    int v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(theirs) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(theirs));
    return v;
}

// counts[warp][E] and total[E] in dynamic shared memory
__global__ void __launch_bounds__(SORT_THREADS) expert_sort_kernel(const int *idx, int n, int E, int ctas, int *order, int *place, int *offsets,
                                                                   W4Slots slots)
{
    extern __shared__ int sm[];
    int *count = sm, *total = sm + SORT_WARPS * E;
    __shared__ int s_part[2][SORT_WARPS], s_valid[SORT_WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = ctas > 1 ? (int)cluster_cta_rank() : 0;
    // this warp's picks: a multiple of 32 of them
    const int share = (n + ctas * SORT_WARPS * 32 - 1) / (ctas * SORT_WARPS * 32) * 32;
    const long long p0 = (long long)share * (rank * SORT_WARPS + warp), p1 = p0 + share < n ? p0 + share : n;
    int *mine = count + warp * E;
    auto expert_of = [&](long long p) {
        const int e = p < p1 ? __ldg(idx + p) : -1;
        return e >= 0 && e < E ? e : -1;
    };
    // the first picks are asked for together and stay in registers
    int held[SORT_HELD];
#pragma unroll
    for (int i = 0; i < SORT_HELD; i++) held[i] = expert_of(p0 + 32 * i + lane);
    for (int e = lane; e < E; e += 32) mine[e] = 0;
    __syncwarp();
    auto rounds = [&](auto &&step) {
#pragma unroll
        for (int i = 0; i < SORT_HELD; i++)
            if (p0 + 32 * i < p1) step(p0 + 32 * i, held[i]);
        for (long long p = p0 + 32 * SORT_HELD; p < p1; p += 32) step(p, expert_of(p + lane));
    };
    rounds([&](long long, int e) {
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
    });
    __syncthreads();
    // places of the warps within the CTA, and the CTA's sum
    for (int e = tid; e < E; e += SORT_THREADS) {
        int sum = 0, c[SORT_WARPS];
#pragma unroll
        for (int w = 0; w < SORT_WARPS; w++) c[w] = count[w * E + e];
#pragma unroll
        for (int w = 0; w < SORT_WARPS; w++) { count[w * E + e] = sum; sum += c[w]; }
        total[e] = sum;
    }
    if (ctas > 1) { cluster_arrive(); cluster_wait(); } else __syncthreads();
    // experts e0 and e0 + 1: their picks in the CTAs before this one, and in all
    const int e0 = 2 * tid;
    int before[2] = {0, 0}, all[2] = {0, 0};
    for (int i = 0; i < 2; i++)
        if (e0 + i < E)
            if (ctas == 1) all[i] = total[e0 + i];
            else {
                int c[SORT_CLUSTER];                            // (asked for together)
#pragma unroll
                for (int r = 0; r < SORT_CLUSTER; r++) c[r] = ld_cluster_s32(total + e0 + i, (uint32_t)r);
#pragma unroll
                for (int r = 0; r < SORT_CLUSTER; r++) {
                    all[i] += c[r];
                    if (r < rank) before[i] += c[r];
                }
            }
    // sums over the experts: of the picks, and of the tiles they make
    int rows = slots.n ? slots.rows : 1, here = 0;
    bool many = false;
    if (slots.n && slots.many_rows) {
        const int mine_here = __reduce_add_sync(0xffffffffu, all[0] + all[1]);
        if (lane == 0) s_valid[warp] = mine_here;
        __syncthreads();
        for (int w = 0; w < SORT_WARPS; w++) here += s_valid[w];
        many = here > slots.few_most;
        if (many) rows = slots.many_rows;
    }
    const int tiles[2] = {(all[0] + rows - 1) / rows, (all[1] + rows - 1) / rows};
    int sum = all[0] + all[1], tsum = tiles[0] + tiles[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, sum, o), b = __shfl_up_sync(0xffffffffu, tsum, o);
        if (lane >= o) { sum += a; tsum += b; }
    }
    if (lane == 31) { s_part[0][warp] = sum; s_part[1][warp] = tsum; }
    __syncthreads();
    for (int w = 0; w < warp; w++) { sum += s_part[0][w]; tsum += s_part[1][w]; }
    int first[2], tile[2];
    first[0] = sum - all[0] - all[1]; first[1] = first[0] + all[0];
    tile[0] = tsum - tiles[0] - tiles[1]; tile[1] = tile[0] + tiles[0];
    if (ctas > 1) { cluster_arrive(); cluster_wait(); }        // every CTA has read every total
    for (int i = 0; i < 2; i++) {
        if (e0 + i >= E) continue;
        total[e0 + i] = first[i] + before[i];                   // this CTA's first place of the expert
        if (rank == 0) {
            offsets[e0 + i] = first[i];
            if (e0 + i == E - 1) offsets[E] = first[i] + all[i];
            if (slots.n) {
                for (int k = 0; k < tiles[i]; k++) {
                    slots.expert[tile[i] + k] = e0 + i;
                    slots.first[tile[i] + k] = first[i] + k * rows;
                    slots.count[tile[i] + k] = min(rows, all[i] - k * rows);
                }
                if (e0 + i == E - 1) {
                    slots.n[0] = many ? 0 : tile[i] + tiles[i];
                    if (slots.many_rows) { slots.n[1] = many ? tile[i] + tiles[i] : 0; slots.n[2] = many ? here : 0; }
                }
            }
        }
    }
    __syncthreads();
    int valid = 0;
    for (int w = 0; w < SORT_WARPS; w++) valid += s_part[0][w];
    rounds([&](long long p, int e) {
        const uint32_t same = __match_any_sync(0xffffffffu, e), below = same & ((1u << lane) - 1u);
        int at = -1;
        if (e >= 0) at = total[e] + mine[e] + __popc(below);
        __syncwarp();
        if (e >= 0 && !below) mine[e] += __popc(same);
        __syncwarp();
        if (p + lane < p1) {
            place[p + lane] = at;
            if (at >= 0) order[at] = (int)(p + lane);
            if (p + lane >= valid) order[p + lane] = -1;
        }
    });
}

int expert_sort(cudaStream_t st, const int *idx, int T, int topk, int E, int *order, int *place, int *offsets, const W4Slots *slots)
{
    static SmemGrant grant;
    const int n = T * topk, ctas = n <= SORT_ALONE ? 1 : SORT_CLUSTER;
    const size_t smem = (size_t)(SORT_WARPS + 1) * E * sizeof(int);
    const W4Slots none{};
    if (!dev_opt_in_smem((const void *)expert_sort_kernel, smem, grant)) return -1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(SORT_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    ++g_launches;
    return cudaLaunchKernelEx(&cfg, expert_sort_kernel, idx, n, E, ctas, order, place, offsets, slots ? *slots : none) == cudaSuccess ? 0 : -1;
}

// Rows one after the other by CTAs that fill the GPU once (a CTA for each of 16384 picks, of which 2048 were here, took 14 us). PIECE:
// bytes of one load, four of which a thread has on their way.
template <typename PIECE>
__global__ void __launch_bounds__(256) expert_gather_kernel(const uint8_t *x, size_t row_bytes, size_t ldx, size_t ldr, const int *order,
                                                            const int *offsets, int picks, int topk, int E, uint8_t *rows)
{
    const int n = min(__ldg(offsets + E), picks), pieces = (int)(row_bytes / sizeof(PIECE));
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int p = __ldg(order + i);
        if (p < 0 || p >= picks) continue;                      // (not an order that the sort wrote)
        const PIECE *src = reinterpret_cast<const PIECE *>(x + (size_t)(p / topk) * ldx);
        PIECE *dst = reinterpret_cast<PIECE *>(rows + (size_t)i * ldr);
        for (int c0 = threadIdx.x; c0 < pieces; c0 += 1024) {
            PIECE v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) if (c0 + 256 * k < pieces) v[k] = __ldg(src + c0 + 256 * k);
#pragma unroll
            for (int k = 0; k < 4; k++) if (c0 + 256 * k < pieces) dst[c0 + 256 * k] = v[k];
        }
    }
}

void expert_gather(cudaStream_t st, const void *x, size_t row_bytes, size_t x_bytes, size_t out_bytes, const int *order, const int *offsets,
                   int n, int topk, int E, void *rows)
{
    const size_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows) | row_bytes | x_bytes | out_bytes;
    const uint8_t *src = static_cast<const uint8_t *>(x);
    uint8_t *dst = static_cast<uint8_t *>(rows);
    const int grid = n < 8 * dev_sms() ? n : 8 * dev_sms();
    if (all % 16 == 0) G5B_LAUNCH(expert_gather_kernel<uint4>, grid, 256, 0, st, src, row_bytes, x_bytes, out_bytes, order, offsets, n, topk, E, dst);
    else if (all % 4 == 0) G5B_LAUNCH(expert_gather_kernel<uint32_t>, grid, 256, 0, st, src, row_bytes, x_bytes, out_bytes, order, offsets, n, topk, E, dst);
    else G5B_LAUNCH(expert_gather_kernel<uint16_t>, grid, 256, 0, st, src, row_bytes, x_bytes, out_bytes, order, offsets, n, topk, E, dst);
}

__device__ __forceinline__ float row_value(const float *p) { return *p; }
__device__ __forceinline__ float row_value(const uint16_t *p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void row_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void row_store(uint16_t *p, float v) { *p = __bfloat16_as_ushort(__float2bfloat16_rn(v)); }

// A CTA: one token, up to 256 * V * CH columns. V values of a row are one load, CH of which a thread has on their way for each pick.
template <typename IN, typename OUT, int V, int CH>
__global__ void __launch_bounds__(256) expert_combine_kernel(const IN *rows, size_t ldr, const int *place, int E, const float *w, int topk, int cols,
                                                             OUT *out, size_t ldo)
{
    __shared__ int s_at[G5B_MAX_TOPK];
    __shared__ float s_w[G5B_MAX_TOPK];
    pdl_wait();
    struct __align__(sizeof(IN) * V) InV { IN v[V]; };
    struct __align__(sizeof(OUT) * V) OutV { OUT v[V]; };
    const int t = blockIdx.x, c0 = (blockIdx.y * 256 * CH + threadIdx.x) * V;
    if (threadIdx.x < topk) {
        int p = load_new(place + (size_t)t * topk + threadIdx.x);
        if (E) p = p >= 0 && p < E ? t * topk + (int)threadIdx.x : -1;
        else if (p >= (int)gridDim.x * topk) p = -1;            // (not a place that the sort wrote)
        s_at[threadIdx.x] = p;
        s_w[threadIdx.x] = w ? __ldg(w + (size_t)t * topk + threadIdx.x) : 1.0f;
    }
    __syncthreads();
    float sum[CH][V];
#pragma unroll
    for (int q = 0; q < CH; q++)
#pragma unroll
        for (int i = 0; i < V; i++) sum[q][i] = 0.f;
#pragma unroll 2
    for (int k = 0; k < topk; k++) {
        const int p = s_at[k];
        if (p < 0) continue;
        const float f = s_w[k];
        const IN *row = rows + (size_t)p * ldr + c0;
        InV in[CH];
#pragma unroll
        for (int q = 0; q < CH; q++) if (c0 + q * 256 * V < cols) in[q] = *reinterpret_cast<const InV *>(row + q * 256 * V);
#pragma unroll
        for (int q = 0; q < CH; q++)
#pragma unroll
            for (int i = 0; i < V; i++) sum[q][i] = fmaf(f, row_value(&in[q].v[i]), sum[q][i]);
    }
#pragma unroll
    for (int q = 0; q < CH; q++) {
        if (c0 + q * 256 * V >= cols) continue;
        OutV o;
#pragma unroll
        for (int i = 0; i < V; i++) row_store(&o.v[i], sum[q][i]);
        *reinterpret_cast<OutV *>(out + (size_t)t * ldo + c0 + q * 256 * V) = o;
    }
}

template <typename IN, typename OUT>
static void combine_as(cudaStream_t st, const void *rows, size_t ldr, const int *place, int E, const float *w, int T, int topk, int cols, void *out, size_t ldo, bool early)
{
    constexpr int V = 16 / (sizeof(IN) > sizeof(OUT) ? sizeof(IN) : sizeof(OUT));
    const IN *in = static_cast<const IN *>(rows);
    OUT *o = static_cast<OUT *>(out);
    const bool wide = reinterpret_cast<uintptr_t>(rows) % (V * sizeof(IN)) == 0 && reinterpret_cast<uintptr_t>(out) % (V * sizeof(OUT)) == 0 &&
                      ldr % V == 0 && ldo % V == 0 && cols % V == 0;
    // few tokens: a load a thread and pick, so that more CTAs share a row
    auto launch = [&](auto v, auto ch) {
        constexpr int W = decltype(v)::value, CH = decltype(ch)::value;
        const dim3 grid(T, (cols + 256 * W * CH - 1) / (256 * W * CH));
        if (early) G5B_LAUNCH_PDL((expert_combine_kernel<IN, OUT, W, CH>), grid, dim3(256), 0, st, in, ldr, place, E, w, topk, cols, o, ldo);
        else       G5B_LAUNCH((expert_combine_kernel<IN, OUT, W, CH>), grid, 256, 0, st, in, ldr, place, E, w, topk, cols, o, ldo);
    };
    using std::integral_constant;
    if (!wide) launch(integral_constant<int, 1>(), integral_constant<int, 1>());
    else if (T <= 256) launch(integral_constant<int, V>(), integral_constant<int, 1>());
    else launch(integral_constant<int, V>(), integral_constant<int, 16 / V>());
}

void expert_combine(cudaStream_t st, const void *rows, int rows_dt, size_t ldr, const int *place, int E, const float *w, int T, int topk, int cols,
                    void *out, int out_dt, size_t ldo, bool early)
{
    if (rows_dt == DT_F32 && out_dt == DT_F32) combine_as<float, float>(st, rows, ldr, place, E, w, T, topk, cols, out, ldo, early);
    else if (rows_dt == DT_F32)                combine_as<float, uint16_t>(st, rows, ldr, place, E, w, T, topk, cols, out, ldo, early);
    else                                       combine_as<uint16_t, uint16_t>(st, rows, ldr, place, E, w, T, topk, cols, out, ldo, early);
}

}  // namespace g5b
