// Around the products of ragged groups: the (row, choice) pairs of a step in the order of the experts they ask (group_rows), and of every row's
// answers the sum with the router's weights (combine_groups).
//
// group_rows is a stable counting sort of pairs by expert, in ONE launch: a cluster of up to eight blocks, every warp a run of neighbouring pairs.
// (1) a warp counts its run's experts, 32 pairs at a time (lanes of the same expert find one another, the first of them adds their number: no
// atomics, and the order is the pairs'); (2) the counts of a block's warps, then of the cluster's blocks (through distributed shared memory), then
// of the experts in front become each warp's first place for each expert; (3) a warp walks its run again and places its pairs. Latency bounds it: two
// walks over what is in L2, three meetings.
//
// combine_groups reads every answer once and writes every row once: memory bounds it. The sum runs over a row's choices in their order in float32,
// whatever place the pairs have: equal bits in every batch.
#include "common.cuh"
#include "fp8_view.h"
#include "tcgen05_common.cuh"

namespace {

constexpr int MAX_GROUPS = 1024, MOST_WARPS = 32;

__device__ __forceinline__ int of_block(const int* p, uint32_t rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(tc::in_block(tc::smem_u32(p), rank)) : "memory");
    return v;
}

// `run`: pairs of a warp, a multiple of 32. Shared memory: counts [warps][groups], then the block's [groups].
__global__ void __launch_bounds__(MOST_WARPS * 32) group_rows_kernel(const int* __restrict__ choice, int ld, int top, long long pairs, int groups, int run, int* __restrict__ offsets,
                                                                     int* __restrict__ order, int* __restrict__ place) {
    extern __shared__ int counts[];
    __shared__ int sums[MOST_WARPS + 1];
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, blocks = gridDim.x, rank = blockIdx.x;
    int *mine = counts + warp * groups, *block_count = counts + warps * groups;
    for (int i = threadIdx.x; i < warps * groups; i += blockDim.x) counts[i] = 0;
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    const long long first = ((long long)rank * warps + warp) * run, end = first + run < pairs ? first + run : pairs;
    auto expert = [&](long long p) {
        if (p >= end) return -1;
        int row, c;
        split_item(p, top, row, c);
        const int e = choice[(size_t)row * ld + c];
        return e >= 0 && e < groups ? e : -1;
    };
    for (long long p = first + lane; p - lane < end; p += 32) {
        const int e = expert(p);
        const unsigned same = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && (same & ((1u << lane) - 1u)) == 0) mine[e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    // a warp's first place among its block's pairs of an expert, and the block's count
    for (int e = threadIdx.x; e < groups; e += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < warps; ++w) {
            const int c = counts[w * groups + e];
            counts[w * groups + e] = sum;
            sum += c;
        }
        block_count[e] = sum;
    }
    __syncthreads();
    if (blocks > 1) {
        tc::cluster_arrive();
        tc::cluster_wait();
    }
    // the experts in front: thread t has `each` neighbouring experts
    const int each = (groups + blockDim.x - 1) / blockDim.x, e0 = min((int)threadIdx.x * each, groups), e1 = min(e0 + each, groups);
    int total = 0;
    for (int e = e0; e < e1; ++e) {
        int all = 0;
        for (int b = 0; b < blocks; ++b) all += of_block(block_count + e, b);
        total += all;
    }
    int upto = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int left = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += left;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    if (warp == 0) {
        const int s = lane < warps ? sums[lane] : 0;
        int run_sum = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, run_sum, o);
            if (lane >= o) run_sum += left;
        }
        if (lane < warps) sums[lane] = run_sum - s;
        if (lane == 31) sums[MOST_WARPS] = run_sum;
    }
    __syncthreads();
    int at = sums[warp] + upto - total;
    for (int e = e0; e < e1; ++e) {
        if (rank == 0) offsets[e] = at;
        int below = 0, all = 0;
        for (int b = 0; b < blocks; ++b) {
            const int c = of_block(block_count + e, b);
            if (b < rank) below += c;
            all += c;
        }
        for (int w = 0; w < warps; ++w) counts[w * groups + e] += at + below;
        at += all;
    }
    const int routed = sums[MOST_WARPS];
    if (rank == 0 && threadIdx.x == 0) offsets[groups] = routed;
    __syncthreads();
    for (long long p = first + lane; p - lane < end; p += 32) {
        const int e = expert(p);
        const unsigned same = __match_any_sync(0xffffffffu, e);
        int to = -1;
        if (e >= 0) to = mine[e] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e >= 0 && (same & ((1u << lane) - 1u)) == 0) mine[e] += __popc(same);
        __syncwarp();
        if (p < end) {
            place[p] = to;
            if (to >= 0) order[to] = (int)p;
        }
    }
    // the pairs without an expert leave the end of the order empty
    for (long long p = routed + (long long)rank * blockDim.x + threadIdx.x; p < pairs; p += (long long)blocks * blockDim.x) order[p] = -1;
    if (blocks > 1) {          // (nobody's counts are gone while others read them)
        tc::cluster_arrive();
        tc::cluster_wait();
    }
}

// A thread has 16 bytes of answers (PER values) of a row; `vec`: 16-byte accesses are allowed.
template <typename Ta, typename Tout, int PER>
__global__ void __launch_bounds__(256) combine_groups_kernel(const Ta* __restrict__ answers, int lda, const int* __restrict__ place, const float* __restrict__ share, int ld_share, int top,
                                                             Tout* __restrict__ out, int ldo, int rows, int cols, int pieces, bool add) {
    pdl_wait();
    pdl_trigger();
    const long long items = (long long)rows * pieces;
    for (long long item = (long long)blockIdx.x * 256 + threadIdx.x; item < items; item += (long long)gridDim.x * 256) {
        int row, piece;
        split_item(item, pieces, row, piece);
        const int c0 = piece * PER;
        float sum[PER];
#pragma unroll
        for (int q = 0; q < PER; ++q) sum[q] = 0.f;
        constexpr int TOGETHER = 4;
        for (int j = 0; j < top; j += TOGETHER) {
            __align__(16) Ta v[TOGETHER][PER];
            float w[TOGETHER];
            bool there[TOGETHER];
#pragma unroll
            for (int i = 0; i < TOGETHER; ++i) {
                there[i] = false;
                if (j + i >= top) continue;
                const int p = place[(size_t)row * top + j + i];
                there[i] = p >= 0;
                if (!there[i]) continue;
                w[i] = share[(size_t)row * ld_share + j + i];
                const Ta* src = answers + (size_t)p * lda + c0;
                if constexpr (PER > 1) *reinterpret_cast<uint4*>(v[i]) = *reinterpret_cast<const uint4*>(src);
                else v[i][0] = src[0];
            }
#pragma unroll
            for (int i = 0; i < TOGETHER; ++i)
                if (there[i])
#pragma unroll
                    for (int q = 0; q < PER; ++q) sum[q] = __fmaf_rn(w[i], to_float(v[i][q]), sum[q]);
        }
        Tout* dst = out + (size_t)row * ldo + c0;
        constexpr int BYTES = PER * (int)sizeof(Tout);
        __align__(16) Tout o[PER];
        if (add) {
            if constexpr (BYTES >= 16)
#pragma unroll
                for (int b = 0; b < BYTES / 16; ++b) reinterpret_cast<uint4*>(o)[b] = reinterpret_cast<const uint4*>(dst)[b];
            else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(dst);
            else o[0] = dst[0];
#pragma unroll
            for (int q = 0; q < PER; ++q) sum[q] = __fadd_rn(to_float(o[q]), sum[q]);
        }
#pragma unroll
        for (int q = 0; q < PER; ++q) o[q] = from_float<Tout>(sum[q]);
        if constexpr (BYTES >= 16)
#pragma unroll
            for (int b = 0; b < BYTES / 16; ++b) reinterpret_cast<uint4*>(dst)[b] = reinterpret_cast<const uint4*>(o)[b];
        else if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
        else dst[0] = o[0];
    }
}

template <typename Ta, typename Tout>
int combine(const void* answers, int lda, const RowGroupsView* g, const float* share, int ld_share, void* out, int ldo, int cols, bool add, cudaStream_t stream) {
    constexpr int PER = 16 / sizeof(Ta);
    const bool vec = ((uintptr_t)answers % 16) == 0 && ((uintptr_t)out % 16) == 0 && (size_t)lda * sizeof(Ta) % 16 == 0 && (size_t)ldo * sizeof(Tout) % 16 == 0 && cols % PER == 0;
    const int pieces = vec ? cols / PER : cols;
    const long long all = ((long long)g->rows * pieces + 255) / 256, most = (long long)jllm_device_sm_count() * 16;
    const dim3 grid((unsigned)(all < most ? all : most));
    if (vec)
        jllm_launch(combine_groups_kernel<Ta, Tout, PER>, grid, dim3(256), 0, stream, LAUNCH_DEPENDENT, static_cast<const Ta*>(answers), lda, (const int*)g->place, share, ld_share,
                    g->top, static_cast<Tout*>(out), ldo, g->rows, cols, pieces, add);
    else
        jllm_launch(combine_groups_kernel<Ta, Tout, 1>, grid, dim3(256), 0, stream, LAUNCH_DEPENDENT, static_cast<const Ta*>(answers), lda, (const int*)g->place, share, ld_share,
                    g->top, static_cast<Tout*>(out), ldo, g->rows, cols, pieces, add);
    return jllm_check_launch("combine_groups");
}

}  // namespace

// `choice` [rows, top]: a pair's expert, anything outside [0, groups) none. Writes offsets [groups + 1], order [rows x top] (-1 behind the last pair)
// and place [rows x top] (-1: no expert).
JLLM_EXPORT int jllm_group_rows(const int* choice, int ld, const RowGroupsView* g, cudaStream_t stream) {
    const long long pairs = (long long)g->rows * g->top;
    JLLM_REQUIRE(g->rows >= 0 && g->top >= 1 && pairs <= BLOCK_MOST && g->groups >= 1 && g->groups <= MAX_GROUPS && ld >= g->top,
                 "group_rows: %d rows of %d choices (%d apart) among %d groups (1 to %d)", g->rows, g->top, ld, g->groups, MAX_GROUPS);
    // a run of 32 pairs a warp while eight blocks hold them, longer ones beyond
    const long long runs = (pairs + 31) / 32;
    const int blocks = runs <= MOST_WARPS ? 1 : runs <= 2 * MOST_WARPS ? 2 : runs <= 4 * MOST_WARPS ? 4 : 8;
    int warps = runs < MOST_WARPS ? (int)(runs < 1 ? 1 : runs) : MOST_WARPS;
    // (a warp's counts lie in shared memory: 227 KB hold 32 warps of 1,024 groups; few pairs leave few warps to walk many groups)
    if (warps < 8) warps = 8;
    const int run = (int)(((pairs + (long long)blocks * warps - 1) / ((long long)blocks * warps) + 31) / 32 * 32);
    const size_t smem = (size_t)(warps + 1) * g->groups * sizeof(int);
    auto kern = group_rows_kernel;
    if (jllm_allow_smem((const void*)kern, smem) != cudaSuccess) return jllm_fail(JLLM_CUDA_ERROR, "group_rows: %zu bytes of shared memory refused", smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (jllm_launch_overlaps(smem, LAUNCH_DEPENDENT)) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    cudaLaunchKernelEx(&cfg, kern, choice, ld, g->top, pairs, g->groups, run, g->offsets, g->order, g->place);
    return jllm_check_launch("group_rows");
}

JLLM_EXPORT int jllm_combine_groups(const void* answers, int answers_dtype, int lda, const RowGroupsView* g, const float* share, int ld_share, void* out, int out_dtype, int ldo, int cols,
                                    int add, cudaStream_t stream) {
    JLLM_REQUIRE(g->rows >= 0 && g->top >= 1 && cols >= 1 && cols <= BLOCK_MOST && lda >= cols && ldo >= cols && ld_share >= g->top,
                 "combine_groups: %d rows of %d choices (%d apart), %d columns (answers %d, out %d apart)", g->rows, g->top, ld_share, cols, lda, ldo);
    if (g->rows == 0) return JLLM_OK;
    if (answers_dtype == JLLM_F32)
        return out_dtype == JLLM_F32 ? combine<float, float>(answers, lda, g, share, ld_share, out, ldo, cols, add != 0, stream)
                                     : combine<float, __nv_bfloat16>(answers, lda, g, share, ld_share, out, ldo, cols, add != 0, stream);
    return out_dtype == JLLM_F32 ? combine<__nv_bfloat16, float>(answers, lda, g, share, ld_share, out, ldo, cols, add != 0, stream)
                                 : combine<__nv_bfloat16, __nv_bfloat16>(answers, lda, g, share, ld_share, out, ldo, cols, add != 0, stream);
}
