// Around the products of ragged groups: the (row, choice) pairs of a step in the order of the experts they ask (group_rows), and of every row's
// answers the sum with the router's weights (combine_groups).
//
// group_rows is a stable counting sort of pairs by expert. A block has a run of neighbouring pairs and every warp of it a part of the run.
// (1) a warp counts its pairs' experts, 32 pairs at a time (lanes of the same expert find one another by votes on its bits, the first of them adds their
// number: no atomics, and the order is the pairs'), and each pair keeps its number among its warp's of that expert; (2) the warps' counts, and the
// experts' in front, become each warp's first place for each expert; (3) every pair has its place, and the block's pairs leave in their experts' order.
// Up to 2,048 pairs are one block and one launch. Of more, a launch in front counts every block's pairs by expert, and (2) adds up the blocks in front.
// Latency bounds the small ones: 64 pairs of 128 experts 2.2 us, 16,384 6.1, 131,072 of 256 9.6 (a cluster of eight blocks took 23 us for the votes and scattered words
// of 8 SMs).
//
// combine_groups reads every answer once and writes every row once: memory bounds it. The sum runs over a row's choices in their order in float32,
// whatever place the pairs have: equal bits in every batch. 2,048 rows of eight float32 answers of 2,048 values 24.4 to 24.9 us (5.5 TB/s; 23.6 at best), bfloat16 12.1; 16 rows 2.3 us.
#include "common.cuh"
#include "fp8_view.h"

namespace {

constexpr int MAX_GROUPS = 1024, MOST_WARPS = 32, HELD = 2, MOST_BLOCKS = GROUP_BLOCKS;
static_assert(32 * HELD * MOST_WARPS <= 1 << 11 && MAX_GROUPS <= 1 << 10, "a pair and its expert share a word");

__device__ __forceinline__ int expert_of(const int* choice, int ld, int top, int groups, long long p) {
    size_t at = (size_t)p;
    if (ld != top) {
        int row, c;
        split_item(p, top, row, c);
        at = (size_t)row * ld + c;
    }
    const int e = choice[at];
    return e >= 0 && e < groups ? e : -1;
}

// counts[block][expert] of the pairs [block * of_block, ...)
__global__ void __launch_bounds__(1024) count_rows_kernel(const int* __restrict__ choice, int ld, int top, long long pairs, int groups, int of_block, int* __restrict__ counts) {
    __shared__ int mine[MAX_GROUPS];
    for (int e = threadIdx.x; e < groups; e += blockDim.x) mine[e] = 0;
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    const long long first = (long long)blockIdx.x * of_block, end = first + of_block < pairs ? first + of_block : pairs;
    for (long long p = first + threadIdx.x; p < end; p += blockDim.x) {
        const int e = expert_of(choice, ld, top, groups, p);
        if (e >= 0) atomicAdd(&mine[e], 1);          // (sums of whole numbers: their order does not matter)
    }
    __syncthreads();
    for (int e = threadIdx.x; e < groups; e += blockDim.x) counts[(size_t)blockIdx.x * groups + e] = mine[e];
}

// `run`: pairs of a warp, a multiple of 32. Shared memory: counts [warps][groups], the block's first places in the order and in itself and all
// blocks' counts [groups] each, and of runs that are held the block's pairs (11 bits) with their experts (10).
__global__ void __launch_bounds__(MOST_WARPS * 32) group_rows_kernel(const int* __restrict__ choice, int ld, int top, long long pairs, int groups, int run, const int* __restrict__ block_counts,
                                                                     int* __restrict__ offsets, int* __restrict__ order, int* __restrict__ place) {
    extern __shared__ int counts[];
    __shared__ unsigned long long sums[MOST_WARPS + 1];
    static_assert(sizeof(sums) <= 1024, "beside 47 KB in a launch's 48");
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, blocks = gridDim.x, rank = blockIdx.x;
    int *mine = counts + warp * groups, *block_first = counts + warps * groups, *local_first = block_first + groups, *all_of = local_first + groups;
    uint32_t* sorted = reinterpret_cast<uint32_t*>(all_of + groups);
    for (int i = threadIdx.x; i < warps * groups; i += blockDim.x) counts[i] = 0;
    pdl_wait();
    pdl_trigger();
    const long long block_at = (long long)rank * warps * run, first = block_at + (long long)warp * run, end = first + run < pairs ? first + run : pairs;
    auto expert = [&](long long p) { return p < end ? expert_of(choice, ld, top, groups, p) : -1; };
    const bool held = run <= 32 * HELD;
    int e_of[HELD], number[HELD];
    if (held)
#pragma unroll
        for (int i = 0; i < HELD; ++i) e_of[i] = 32 * i < run ? expert(first + 32 * i + lane) : -1;
    __syncthreads();
    // the 32 pairs' numbers among the warp's of their experts so far
    auto count = [&](int e) {
        unsigned same = __ballot_sync(0xffffffffu, e >= 0);          // (lanes without an expert do not count)
        for (int bit = 1; bit < groups; bit <<= 1) {
            const unsigned set = __ballot_sync(0xffffffffu, e & bit);
            same &= e & bit ? set : ~set;
        }
        const int before = __popc(same & ((1u << lane) - 1u)), so_far = e >= 0 ? mine[e] : 0;
        __syncwarp();
        if (e >= 0 && before == 0) mine[e] = so_far + __popc(same);
        __syncwarp();
        return so_far + before;
    };
    if (held) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (32 * i < run) number[i] = count(e_of[i]);
    } else {
        for (long long p = first + lane; p - lane < end; p += 32) count(expert(p));
    }
    __syncthreads();
    // thread t has `each` neighbouring experts: the warps' counts become their first numbers in the block, and (two sums in one: all blocks' pairs above, the
    // block's below) the experts in front are added up
    const int each = (groups + blockDim.x - 1) / blockDim.x, e0 = min((int)threadIdx.x * each, groups), e1 = min(e0 + each, groups);
    unsigned long long total = 0;
    for (int e = e0; e < e1; ++e) {
        int here = 0;
        for (int w = 0; w < warps; w += 8) {          // (a multiple of eight warps)
            int c[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i] = counts[(w + i) * groups + e];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                counts[(w + i) * groups + e] = here;
                here += c[i];
            }
        }
        int all = here, below = 0;
        if (blocks > 1) {
            all = 0;
#pragma unroll 8
            for (int b = 0; b < blocks; ++b) {
                const int c = block_counts[(size_t)b * groups + e];
                all += c;
                below += b < rank ? c : 0;
            }
        }
        block_first[e] = below, local_first[e] = here, all_of[e] = all;
        total += (unsigned long long)all << 32 | (unsigned)here;
    }
    unsigned long long upto = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long left = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += left;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    if (warp == 0) {
        const unsigned long long s = lane < warps ? sums[lane] : 0;
        unsigned long long so_far = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long left = __shfl_up_sync(0xffffffffu, so_far, o);
            if (lane >= o) so_far += left;
        }
        if (lane < warps) sums[lane] = so_far - s;
        if (lane == 31) sums[MOST_WARPS] = so_far;
    }
    __syncthreads();
    const unsigned long long in_front = sums[warp] + upto - total;
    int at = (int)(in_front >> 32), in_block = (int)(uint32_t)in_front;
    for (int e = e0; e < e1; ++e) {
        if (rank == 0) offsets[e] = at;
        const int here = local_first[e];
        block_first[e] += at, local_first[e] = in_block;
        at += all_of[e], in_block += here;
    }
    const int routed = (int)(sums[MOST_WARPS] >> 32), routed_here = (int)(uint32_t)sums[MOST_WARPS];
    if (rank == 0 && threadIdx.x == 0) offsets[groups] = routed;
    __syncthreads();
    if (held) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (32 * i < run) {
                const long long p = first + 32 * i + lane;
                const int e = e_of[i], n = e >= 0 ? mine[e] + number[i] : 0;
                if (p < end) place[p] = e >= 0 ? block_first[e] + n : -1;
                if (e >= 0) sorted[local_first[e] + n] = (uint32_t)(p - block_at) | (uint32_t)e << 11;
            }
        __syncthreads();
        for (int i = threadIdx.x; i < routed_here; i += blockDim.x) {
            const int e = (int)(sorted[i] >> 11);
            order[block_first[e] + i - local_first[e]] = (int)(block_at + (sorted[i] & 0x7ffu));
        }
    } else {
        // (the counts have become first numbers: counting on from them gives the pairs theirs)
        for (long long p = first + lane; p - lane < end; p += 32) {
            const int e = expert(p), n = count(e);
            if (p < end) {
                place[p] = e >= 0 ? block_first[e] + n : -1;
                if (e >= 0) order[block_first[e] + n] = (int)p;
            }
        }
    }
    // the pairs without an expert leave the end of the order empty
    for (long long p = routed + (long long)rank * blockDim.x + threadIdx.x; p < pairs; p += (long long)blocks * blockDim.x) order[p] = -1;
}

// A thread has 16 bytes of answers (PER values) of a row; `vec`: 16-byte accesses are allowed.
template <typename Ta, typename Tout, int PER>
__global__ void __launch_bounds__(256) combine_groups_kernel(const Ta* __restrict__ answers, int lda, const int* __restrict__ place, const float* __restrict__ share, int ld_share, int top,
                                                             Tout* __restrict__ out, int ldo, int rows, int cols, int pieces, bool add) {
    const unsigned pairs = (unsigned)rows * (unsigned)top;          // (a place of a larger step, not filled anew, is none)
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
                there[i] = (unsigned)p < pairs;
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
    // 32 or 64 pairs a warp while MOST_BLOCKS blocks hold them, longer runs beyond
    constexpr int FULL = 32 * HELD * MOST_WARPS;
    const int blocks = pairs <= FULL ? 1 : pairs <= (long long)FULL * MOST_BLOCKS ? (int)((pairs + FULL - 1) / FULL) : MOST_BLOCKS;
    const int warps = pairs <= 8 * 32 ? 8 : pairs <= 16 * 32 ? 16 : MOST_WARPS;
    const int run = (int)(((pairs + (long long)blocks * warps - 1) / ((long long)blocks * warps) + 31) / 32 * 32);
    const size_t smem = ((size_t)(warps + 3) * g->groups + (run <= 32 * HELD ? (size_t)warps * run : 0)) * sizeof(int);
    // (a launch has 48 KB without asking, of which the kernel holds some hundred bytes by itself)
    if (smem > 47 * 1024 && jllm_allow_smem((const void*)group_rows_kernel, smem) != cudaSuccess)
        return jllm_fail(JLLM_CUDA_ERROR, "group_rows: %zu bytes of shared memory refused", smem);
    if (blocks > 1) {
        JLLM_REQUIRE(g->counts, "group_rows: no room for the blocks' counts");
        jllm_launch(count_rows_kernel, dim3(blocks), dim3(1024), 0, stream, LAUNCH_DEPENDENT, choice, ld, g->top, pairs, g->groups, warps * run, g->counts);
        const int rc = jllm_check_launch("group_rows");
        if (rc != JLLM_OK) return rc;
    }
    jllm_launch(group_rows_kernel, dim3(blocks), dim3(warps * 32), smem, stream, LAUNCH_DEPENDENT, choice, ld, g->top, pairs, g->groups, run, (const int*)g->counts, g->offsets, g->order,
                g->place);
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
