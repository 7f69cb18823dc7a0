// out[m, n] (+)= (sum_k qa[m, k] * qw[n, k]) * scale_a[m] * scale_w[n] (+ bias[n]), 8-bit integers with one scale a token and one a
// weight row, on the 5th-generation tensor cores (kind::i8). The sum is exact in 32-bit integers (k up to 131,071: 131,071 * 128 * 128 <
// 2^31), so its order does not matter: every way of cutting the work gives the same bits, and a row's result does not depend on what else
// is in the batch.
//
// The weight is PACKED once (ops.pack_int8): tiles of 128 rows x 128 k, each the 16 KB image that the tensor cores read from shared
// memory (rows of 128 bytes, 16-byte chunk c of row r at chunk position c ^ (r & 7): the 128-byte swizzle), tile (t, kb) at (t *
// k_blocks + kb) * 16 KB; its scales are filled up to whole tiles. The activations' tiles come by tiled TMA copies, which fill rows
// beyond M and k beyond K with zeros.
//
// Two kernels. Few tokens (`swap`): the weight rows are the M side of the MMAs, the tokens the N side, and a cluster of blocks shares the
// k blocks of 128 weight rows. Many tokens (`pair`): two SMs to a tile of 256 tokens x 64, 128 or 256 weight rows. Every wait is bounded
// and raises the products' error word (codes 31-33 swap, 34-36 pair).
#include "gemm_epilogue.cuh"
#include "int8_view.h"

namespace {

using namespace tc;

constexpr int BK = 128, TILE_BYTES = 128 * BK;
constexpr int MAX_K = 131071;
constexpr int THREADS = 192;           // warp 0 producer, warp 1 MMA, warps 2..5 epilogue
constexpr size_t SMEM_ROOM = 224 * 1024;

// kind::i8: 32-bit integer accumulators, A and B signed 8-bit, both K-major
__host__ __device__ constexpr uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// the address, in the cluster's shared window, of `addr` (an address in this block's shared memory) in block `rank`
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

// The result from the exact sum: the same operations in the same order in both kernels.
__device__ __forceinline__ float scaled(uint32_t sum, float scale_a, float scale_w) {
    return __fmul_rn(__fmul_rn((float)(int)sum, scale_a), scale_w);
}

// ---- few tokens: a cluster of blocks to 128 weight rows --------------------------------------------------------------------
// With few tokens the product is nothing but reading W once. Block p of a cluster streams its part of the tile's k blocks (one contiguous
// 16 KB bulk copy each, requested before the kernel in front has finished: weights are nobody's output); the accumulator [128 weight
// rows x tokens] lies in its tensor memory. Of the tokens every block finishes a share: the others send their parts of it (st.async,
// which counts its bytes on the owner's mbarrier: one way through the cluster and no meeting), the owner adds them up, scales and stores.
struct SwapArgs {
    const int8_t* w;
    const float *scale_w, *scale_a;
    VecRef bias;
    int has_bias, ldo, accumulate, M, N, k_blocks, ntok, stages, blocks, share;      // ntok: the MMAs' N; share: tokens a block finishes
    uint32_t tmem_cols;
    GluArgs glu;
    int* error_word;
};

__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((i & 1023u) == 1023u && *abort_flag) return false;
    }
    return false;
}

template <typename Tout>
__global__ void __launch_bounds__(THREADS, 1)
gemm_int8_swap_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ SwapArgs g, Tout* __restrict__ out) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(16) float token_scales[256];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* aligned = smem_raw + (base - smem_u32(smem_raw));
    const int stages = g.stages, blocks = g.blocks, share = g.share;
    const uint32_t stage_bytes = TILE_BYTES + (uint32_t)g.ntok * BK, parts_at = (uint32_t)stages * stage_bytes;
    const uint32_t part_bytes = (uint32_t)share * 128 * 4;         // one block's part of a share, [share / 4][128 rows][4 tokens]
    const uint32_t bars_at = parts_at + (uint32_t)(blocks - 1) * part_bytes, bars = base + bars_at;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (stages + s); };
    const uint32_t acc_bar = bars + 16u * stages, parts_bar = acc_bar + 8u;
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(aligned + bars_at + 8 * (2 * stages + 2));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int tile = (int)blockIdx.x / blocks, rank = (int)blockIdx.x % blocks;      // (clusters lie along x: this is the rank)
    const int kb_lo = (int)((long long)g.k_blocks * rank / blocks), n_kb = (int)((long long)g.k_blocks * (rank + 1) / blocks) - kb_lo;
    const int tokens = (g.M + 7) & ~7;                              // the accumulator's columns that anybody needs
    const int mine = rank * share, mine_end = min(mine + share, tokens);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(acc_bar, 1);
        mbar_init(parts_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        mbar_expect_tx(parts_bar, (uint32_t)(blocks - 1) * (uint32_t)max(0, mine_end - mine) * 512u);
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)), "r"(g.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_base_slot;
    if (blocks > 1) cluster_arrive();          // (waited for in front of the first send: every block runs and has its barriers)

    bool ok = true;
    if (warp == 0) {
        // ---------------- producer: weights by bulk copy, activations by TMA ----------------
        const int8_t* w = g.w + ((size_t)tile * g.k_blocks + kb_lo) * TILE_BYTES;
        const int early = min(stages, n_kb);
        if (elect_one())
            for (int i = 0; i < early; ++i) {
                mbar_expect_tx(full_bar(i), stage_bytes);
                bulk_copy(base + (uint32_t)i * stage_bytes, w + (size_t)i * TILE_BYTES, TILE_BYTES, full_bar(i));
            }
        __syncwarp();
        pdl_wait();
        pdl_trigger();
        if (elect_one())
            for (int i = 0; i < early; ++i)
                tma_load_2d(base + (uint32_t)i * stage_bytes + TILE_BYTES, &map_a, (kb_lo + i) * BK, 0, full_bar(i));
        __syncwarp();
        int s = 0;
        uint32_t parity = 0;                                   // the ring's second lap waits for the first lap's release
        for (int i = stages; i < n_kb; ++i) {
            if (!warp_wait(empty_bar(s), parity, abort_flag)) { ok = false; break; }
            if (elect_one()) {
                const uint32_t dst = base + (uint32_t)s * stage_bytes;
                mbar_expect_tx(full_bar(s), stage_bytes);
                bulk_copy(dst, w + (size_t)i * TILE_BYTES, TILE_BYTES, full_bar(s));
                tma_load_2d(dst + TILE_BYTES, &map_a, (kb_lo + i) * BK, 0, full_bar(s));
            }
            __syncwarp();
            if (++s == stages) { s = 0; parity ^= 1u; }
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicExch(g.error_word, 31); }
        if (blocks > 1) cluster_wait();
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        const uint32_t idesc = idesc_i8(128, g.ntok);
        const uint64_t desc_w0 = smem_desc_sw128(base), desc_b0 = smem_desc_sw128(base + TILE_BYTES);
        uint64_t desc_w = desc_w0, desc_b = desc_b0;          // (a stage further is an addition to the address field)
        int s = 0;
        uint32_t parity = 0;
        for (int i = 0; i < n_kb; ++i) {
            if (!warp_wait(full_bar(s), parity, abort_flag)) { ok = false; break; }
            tcgen05_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < BK / 32; ++k) mma_i8(tmem_base, desc_w + 2 * k, desc_b + 2 * k, idesc, (i > 0 || k > 0) ? 1u : 0u);
                tcgen05_commit(empty_bar(s));
            }
            __syncwarp();
            desc_w += stage_bytes >> 4;
            desc_b += stage_bytes >> 4;
            if (++s == stages) { s = 0; parity ^= 1u; desc_w = desc_w0; desc_b = desc_b0; }
        }
        if (ok) {
            if (elect_one()) tcgen05_commit(acc_bar);
        } else if (lane == 0) { *abort_flag = 1; atomicExch(g.error_word, 32); }
        __syncwarp();
        if (blocks > 1) cluster_wait();
    } else {
        // ---------------- epilogue: warps 2..5, TMEM lanes 32 * (warp % 4) = weight rows of the tile ----------------
        const int quad = warp & 3, row = quad * 32 + lane, n = tile * 128 + row;
        const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16);
        const float sw = g.scale_w[n];                        // (filled up to whole tiles)
        const float b = g.has_bias && n < g.N ? g.bias[n] : 0.f;
        pdl_wait();          // the token scales, and what is added into, were written by the kernels before
        pdl_trigger();
        // (into shared memory while the weights come: asked for in front of every store they were 1 us for 8 tokens)
        for (int i = threadIdx.x - 64; i < 256; i += 128) token_scales[i] = i < g.M ? g.scale_a[i] : 0.f;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (blocks > 1) cluster_wait();
        ok = mbar_wait(acc_bar, 0, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        tcgen05_fence_after();
        if (ok)
            for (int d = 1; d < blocks; ++d) {          // (every block begins with its neighbour: nobody is written by all at once)
                const int p = (rank + d) % blocks, t0 = p * share, t1 = min(t0 + share, tokens);
                // of block p's blocks - 1 parts this block's is number `rank`, or rank - 1 if p is below it
                const uint32_t dst = in_block(base + parts_at + (uint32_t)(rank - (rank > p ? 1 : 0)) * part_bytes + (uint32_t)row * 16, p);
                const uint32_t bar = in_block(parts_bar, p);
                auto send = [&](auto& v, int t) {
                    tmem_ld(taddr + t, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int q = 0; q < (int)(sizeof(v) / 16); ++q)
                        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                                     ::"r"(dst + (uint32_t)((t - t0) / 4 + q) * 2048u), "r"(v[4 * q]), "r"(v[4 * q + 1]), "r"(v[4 * q + 2]),
                                     "r"(v[4 * q + 3]), "r"(bar)
                                     : "memory");
                };
                int t = t0;
                uint32_t v16[16], v8[8];
                for (; t + 16 <= t1; t += 16) send(v16, t);
                if (t < t1) send(v8, t);
            }
        if (ok && blocks > 1 && mine < mine_end) ok = __all_sync(0xffffffffu, wait_cluster(parts_bar, 0, abort_flag));
        if (ok) {
            const uint8_t* parts = aligned + parts_at + (size_t)row * 16;
            // Results leave 16 bytes a lane: a warp parks its 32 weight rows x J tokens in the ring (idle by now: every MMA is done) and takes
            // them back token by token. A lane that stores its own values stores 2 bytes of every token's row, with all that a store costs.
            Tout* park = reinterpret_cast<Tout*>(aligned + (size_t)quad * 4096);
            const int width = g.glu ? 16 : 32, column = g.glu ? (tile * 128 + quad * 32) >> 1 : tile * 128 + quad * 32;
            const bool vec = tile * 128 + quad * 32 + 32 <= g.N && ((uintptr_t)out & 15u) == 0 && (((size_t)g.ldo * sizeof(Tout)) & 15u) == 0;
            auto finish = [&](auto& sum, int t) {
                constexpr int J = sizeof(sum) / 4, PER = 16 / sizeof(Tout);       // tokens; values of a 16-byte piece
                tmem_ld(taddr + t, sum);
                float v[J];
                tmem_ld_wait();
                for (int p = 0; p < blocks - 1; ++p) {
                    const uint8_t* src = parts + (size_t)p * part_bytes + (size_t)((t - mine) / 4) * 2048;
#pragma unroll
                    for (int q = 0; q < J / 4; ++q) {
                        const uint4 x = *reinterpret_cast<const uint4*>(src + q * 2048);
                        sum[4 * q] += x.x, sum[4 * q + 1] += x.y, sum[4 * q + 2] += x.z, sum[4 * q + 3] += x.w;
                    }
                }
#pragma unroll
                for (int j = 0; j < J; j += 4) {
                    const float4 sa = *reinterpret_cast<const float4*>(token_scales + t + j);
                    v[j] = scaled(sum[j], sa.x, sw);
                    v[j + 1] = scaled(sum[j + 1], sa.y, sw);
                    v[j + 2] = scaled(sum[j + 2], sa.z, sw);
                    v[j + 3] = scaled(sum[j + 3], sa.w, sw);
                }
                if (g.glu) {
                    // rows come in blocks of 16, 8 gate rows and the 8 up rows of the same hidden units: the gates' lanes take the first half of
                    // the tokens, the others the second
                    const bool up_lane = lane & 8;
                    float gate[J / 2], up[J / 2], units[J / 2];
#pragma unroll
                    for (int j = 0; j < J / 2; ++j) {
                        const float other = __shfl_xor_sync(0xffffffffu, up_lane ? v[j] : v[J / 2 + j], 8);
                        gate[j] = up_lane ? other : v[j];
                        up[j] = up_lane ? v[J / 2 + j] : other;
                    }
                    glu_units<J / 2>(g.glu.word, [&](int j) { return gate[j]; }, [&](int j) { return up[j]; }, 1.f, units);
#pragma unroll
                    for (int j = 0; j < J / 2; ++j)
                        park[(up_lane ? J / 2 + j : j) * 16 + (lane >> 4) * 8 + (lane & 7)] = from_float<Tout>(units[j]);
                } else {
                    if (g.has_bias)
#pragma unroll
                        for (int j = 0; j < J; ++j) v[j] = __fadd_rn(v[j], b);
                    if (g.accumulate == EPI_RELU2)
#pragma unroll
                        for (int j = 0; j < J; ++j) v[j] = epilogue_act(v[j], EPI_RELU2);
                    if (g.accumulate == EPI_ADD) {
                        // (all the old values are requested before the first store: a load behind a store through the same pointer would wait)
                        float old[J];
#pragma unroll
                        for (int j = 0; j < J; ++j) old[j] = n < g.N && t + j < g.M ? to_float(out[(size_t)(t + j) * g.ldo + n]) : 0.f;
#pragma unroll
                        for (int j = 0; j < J; ++j) v[j] = __fadd_rn(v[j], old[j]);
                    }
#pragma unroll
                    for (int j = 0; j < J; ++j) park[j * 32 + lane] = from_float<Tout>(v[j]);
                }
                __syncwarp();
                if (vec) {
                    const int pieces = width / PER;              // of a token's row: 2, 4 or 8
                    for (int i = lane; i < J * pieces; i += 32) {
                        const int j = i / pieces, c = i % pieces * PER;
                        if (t + j < g.M)
                            *reinterpret_cast<uint4*>(out + (size_t)(t + j) * g.ldo + column + c) = *reinterpret_cast<const uint4*>(park + j * width + c);
                    }
                } else {
                    const int last = g.glu ? g.N >> 1 : g.N;
                    for (int i = lane; i < J * width; i += 32) {
                        const int j = i / width, c = i % width;
                        if (t + j < g.M && column + c < last) out[(size_t)(t + j) * g.ldo + column + c] = park[i];
                    }
                }
                __syncwarp();
            };
            int t = mine;
            uint32_t sum16[16], sum8[8];
#pragma unroll 1
            for (; t + 16 <= mine_end; t += 16) finish(sum16, t);
            if (t < mine_end) finish(sum8, t);
        } else if (lane == 0) { *abort_flag = 1; atomicExch(g.error_word, 33); }
    }
    tcgen05_fence_before();
    __syncthreads();
    if (warp == 2) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(g.tmem_cols) : "memory");
    }
    // A block whose wait ran out stays until the others have left (their waits are bounded) or come here: they may still send to it.
    if (blocks > 1 && *abort_flag) {
        cluster_arrive();
        cluster_wait();
    }
}

struct SwapCut {
    int blocks, share, ntok, stages;
    size_t smem;
};
SwapCut swap_cut(int blocks, int M, int k_blocks) {
    SwapCut c{blocks, ((M + 7) / 8 + blocks - 1) / blocks * 8, (M + 15) / 16 * 16, 0, 0};
    const size_t stage = TILE_BYTES + (size_t)c.ntok * BK, parts = (size_t)(blocks - 1) * c.share * 512;
    const size_t room = c.ntok <= 64 ? 104 * 1024 : SMEM_ROOM - 4096;
    c.stages = parts + 2 * stage > room ? 0 : (int)((room - parts) / stage);
    const int most = (k_blocks + blocks - 1) / blocks;
    if (c.stages > most) c.stages = most;
    c.smem = c.stages * stage + parts + 1024 + 8 * (2 * c.stages + 2) + 16;
    return c;
}

// ---- many tokens: two SMs to a tile of 256 tokens x BN weight rows ----------------------------------------------------------
// A cluster of two blocks: each brings 128 tokens and half of the tile's weight rows, one lane of the first block issues MMAs of M 256
// that read both blocks' shared memory, and each block ends up with its 128 tokens in its own tensor memory, where two accumulators let
// a tile's epilogue run under the next tile's main loop. Every copy completes on the FIRST block's "full" barrier of the stage;
// tcgen05.commit, multicast to both blocks, frees the stage in both. The pairs walk the tiles with m fastest.
constexpr int STAGING_BYTES = 4 * STAGING_WARP_FLOATS * 4;
template <int BN> struct PairShape {
    static constexpr int W_BYTES = BN / 2 * BK, STAGE_BYTES = TILE_BYTES + W_BYTES;
    static constexpr int STAGES = 196608 / STAGE_BYTES;
    static constexpr size_t SMEM = (size_t)STAGES * STAGE_BYTES + 1024 + 256 + STAGING_BYTES;
    static_assert(STAGE_BYTES % 1024 == 0 && SMEM <= 227 * 1024, "swizzled tiles lie at multiples of 1,024 bytes");
};

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// a tiled copy into THIS block's shared memory that completes on a barrier that may be the partner's
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t cluster_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(cluster_bar)
        : "memory");
}
// arrives, when the MMAs issued so far are done, on the barrier at this offset in both blocks of the pair
__device__ __forceinline__ void commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3)
                 : "memory");
}

template <typename Tout, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                      const __grid_constant__ CUtensorMap map_out, int bulk_out, const float* __restrict__ scale_a,
                      const float* __restrict__ scale_w, VecRef bias, int has_bias, Tout* __restrict__ out, int ldo, int accumulate, int M,
                      int N, int k_blocks, GluArgs glu, int* __restrict__ error_word) {
    using S = PairShape<BN>;
    constexpr int STAGES = S::STAGES, STAGE_BYTES = S::STAGE_BYTES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* aligned = smem_raw + (base - smem_u32(smem_raw));
    // the stages, the epilogue's staging (1024-byte aligned, as the stages are), the barriers: full[STAGES] (the first block's are used),
    // empty[STAGES] (each block its own), acc_full[2] (each its own), acc_empty[2] (the first block's); then the TMEM base and the abort flag
    const uint32_t bars = base + STAGES * STAGE_BYTES + STAGING_BYTES;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
    auto acc_full_bar = [&](int b) { return bars + 8u * (2 * STAGES + b); };
    auto acc_empty_bar = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(aligned + STAGES * STAGE_BYTES + STAGING_BYTES + 8 * (2 * STAGES + 4));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
    uint8_t* staging = aligned + STAGES * STAGE_BYTES;

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    uint32_t rank;                                    // 0: the pair's first block, which issues the MMAs
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles_m = (M + 255) / 256, tiles = tiles_m * ((N + BN - 1) / BN);
    const int packed_rows = (N + 127) & ~127;         // rows of the packed weight

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full_bar(b), 1);
            mbar_init(acc_empty_bar(b), 8);   // one arrival per epilogue warp of both blocks
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {   // the same warp of both blocks allocates the columns in both
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)), "r"(2 * BN)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();          // the partner's barriers are set up and its tensor memory is there before anything reaches them
    tcgen05_fence_after();
    const uint32_t tmem_base = *tmem_base_slot;
    pdl_wait();
    pdl_trigger();

    auto give_up = [&](int code) {
        *abort_flag = 1;
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(in_block(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1u)), "r"(1) : "memory");
        atomicExch(error_word, code);
    };

    if (warp == 0) {
        // ---------------- producer (both blocks) ----------------
        const uint32_t first_full = in_block(full_bar(0), 0);
        int s = 0;
        uint32_t parity = 1, dst = base;
        bool ok = true;
        for (int tile = pair; ok && tile < tiles; tile += pairs) {
            const int m0 = (tile % tiles_m) * 256 + (int)rank * 128, n0 = (tile / tiles_m) * BN, w0 = n0 + (int)rank * (BN / 2);
            const bool mine = w0 < packed_rows;                            // this block's half of the weight rows exists
            const uint32_t tx = 2 * TILE_BYTES + (n0 + BN / 2 < packed_rows ? 2 : 1) * S::W_BYTES;     // both blocks' bytes
            int wy = (w0 >> 7) * k_blocks * 128 + (w0 & 127);              // row of the packed weight's k block
            for (int kb = 0; kb < k_blocks; ++kb, wy += 128) {
                if (!warp_wait(empty_bar(s), parity, abort_flag)) { ok = false; break; }
                const uint32_t full0 = first_full + 8u * s;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(full_bar(s), tx);
                    tma_load_2d_pair(dst, &map_a, kb * BK, m0, full0);
                    if (mine) tma_load_2d_pair(dst + TILE_BYTES, &map_w, 0, wy, full0);
                }
                __syncwarp();
                dst += STAGE_BYTES;
                if (++s == STAGES) { s = 0; parity ^= 1u; dst = base; }
            }
        }
        if (!ok && lane == 0) give_up(34);
    } else if (warp == 1) {
        // ---------------- MMA issuer (the first block) ----------------
        if (rank == 0) {
            const uint64_t desc_a0 = smem_desc_sw128(base), desc_b0 = smem_desc_sw128(base + TILE_BYTES);
            uint64_t desc_a = desc_a0, desc_b = desc_b0;          // (a stage further is an addition to the address field)
            uint32_t local_tile = 0, parity = 0;
            int s = 0;
            bool ok = true;
            for (int tile = pair; ok && tile < tiles; tile += pairs, ++local_tile) {
                const uint32_t buf = local_tile & 1u;
                if (!warp_wait(acc_empty_bar(buf), ((local_tile >> 1) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
                tcgen05_fence_after();
                const uint32_t tmem_d = tmem_base + buf * BN;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!warp_wait(full_bar(s), parity, abort_flag)) { ok = false; break; }
                    tcgen05_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / 32; ++k)
                            mma_i8_pair(tmem_d, desc_a + 2 * k, desc_b + 2 * k, idesc_i8(256, BN), (kb > 0 || k > 0) ? 1u : 0u);
                        commit_pair(empty_bar(s));          // both blocks' stage is free when these MMAs have read it
                    }
                    __syncwarp();
                    desc_a += STAGE_BYTES >> 4;
                    desc_b += STAGE_BYTES >> 4;
                    if (++s == STAGES) { s = 0; parity ^= 1u; desc_a = desc_a0; desc_b = desc_b0; }
                }
                if (ok && elect_one()) commit_pair(acc_full_bar(buf));
                __syncwarp();
            }
            if (!ok && lane == 0) give_up(35);
        }
    } else {
        // ---------------- epilogue: warps 2..5 of both blocks, TMEM lanes 32 * (warp % 4) ----------------
        const int quad = warp & 3;
        const TileEpilogue<Tout> ep{out, ldo, M, N, accumulate, has_bias, glu, bias, bulk_out ? &map_out : nullptr};
        float* my_staging = reinterpret_cast<float*>(staging + quad * (bulk_out ? BULK_WARP_BYTES : STAGING_WARP_FLOATS * 4));
        uint32_t local_tile = 0;
        bool ok = true;
        for (int tile = pair; ok && tile < tiles; tile += pairs, ++local_tile) {
            const int row0 = (tile % tiles_m) * 256 + (int)rank * 128 + quad * 32, n0 = (tile / tiles_m) * BN;
            const uint32_t buf = local_tile & 1u;
            const float sa = row0 + lane < M ? scale_a[row0 + lane] : 0.f;
            if (!mbar_wait(acc_full_bar(buf), (local_tile >> 1) & 1u, abort_flag)) { ok = false; break; }
            tcgen05_fence_after();
            const uint32_t taddr = tmem_base + buf * BN + ((uint32_t)(quad * 32) << 16);
            const bool whole = ep.rows_whole(row0);
#pragma unroll 1
            for (int c0 = 0; c0 < BN && n0 + c0 < N; c0 += 32) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(taddr + c0, v);
                tmem_ld_wait();
                const float4* sw = reinterpret_cast<const float4*>(scale_w + n0 + c0);      // (filled up to whole tiles)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float4 f = sw[j];
                    v[4 * j] = __float_as_uint(scaled(v[4 * j], sa, f.x));
                    v[4 * j + 1] = __float_as_uint(scaled(v[4 * j + 1], sa, f.y));
                    v[4 * j + 2] = __float_as_uint(scaled(v[4 * j + 2], sa, f.z));
                    v[4 * j + 3] = __float_as_uint(scaled(v[4 * j + 3], sa, f.w));
                }
                ep.store(v, row0, lane, n0 + c0, whole, my_staging);
            }
            tcgen05_fence_before();          // this warp has read the accumulator
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(in_block(acc_empty_bar(buf), 0));
        }
        ep.bulk_done(lane);
        if (!ok && lane == 0) give_up(36);
    }
    tcgen05_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();          // neither block leaves, or frees tensor memory, while the other may still reach into it
    if (warp == 2) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BN) : "memory");
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------

// A [rows, cols] matrix of bytes with row stride ld, read in boxes of box_rows x 128, with the 128-byte swizzle or as it lies.
int byte_map_for(const void* ptr, long long rows, long long cols, long long ld, int box_rows, bool swizzle, CUtensorMap* out) {
    static std::unordered_map<MapKey, CUtensorMap, MapKeyHash> cache;
    static std::mutex mu;
    const MapKey key{ptr, rows, cols, ld, box_rows * 2 + (swizzle ? 1 : 0)};
    std::lock_guard<std::mutex> lock(mu);
    auto it = cache.find(key);
    if (it != cache.end()) {
        *out = it->second;
        return JLLM_OK;
    }
    EncodeTiledFn fn = encode_fn();
    if (!fn) return jllm_fail(JLLM_CUDA_ERROR, "gemm_int8: the driver does not offer cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    CUtensorMap map;
    const CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return jllm_fail(JLLM_CUDA_ERROR, "gemm_int8: cuTensorMapEncodeTiled failed (%d) for [%lld, %lld] bytes, ld %lld", (int)r, rows, cols, ld);
    if (cache.size() > 4096) cache.clear();
    cache.emplace(key, map);
    *out = map;
    return JLLM_OK;
}

template <typename Tout>
int launch_swap(const CUtensorMap& map_a, const SwapArgs& g, const SwapCut& c, int tiles, void* out, cudaStream_t stream) {
    auto kern = gemm_int8_swap_kernel<Tout>;
    if (jllm_allow_smem((const void*)kern, c.smem) != cudaSuccess)
        return jllm_fail(JLLM_CUDA_ERROR, "gemm_int8: %zu bytes of shared memory refused", c.smem);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * c.blocks);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = c.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c.blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (jllm_launch_overlaps(c.smem, LAUNCH_DEPENDENT)) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    cudaLaunchKernelEx(&cfg, kern, map_a, g, static_cast<Tout*>(out));
    return jllm_check_launch("gemm_int8_swap");
}

template <typename Tout, int BN>
int resident_pairs() {
    static int pairs = -1;
    if (pairs >= 0) return pairs;
    auto kern = gemm_int8_pair_kernel<Tout, BN>;
    if (jllm_allow_smem((const void*)kern, PairShape<BN>::SMEM) != cudaSuccess) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * (jllm_device_sm_count() > 0 ? jllm_device_sm_count() : 2));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = PairShape<BN>::SMEM;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    return pairs = n;
}

}  // namespace

int* jllm_gemm_error_word();
extern int g_plain_stores;

namespace {

struct Product {
    const int8_t *a, *w;
    int lda;
    const float *scale_a, *scale_w;
    int k_blocks;
    VecRef bias;
    int has_bias;
    void* out;
    int out_dtype, ldo, accumulate, M, N, K;
    GluArgs glu;
    int* error_word;
    cudaStream_t stream;
};

int run_swap(const Product& p, int blocks) {
    const SwapCut c = swap_cut(blocks, p.M, p.k_blocks);
    JLLM_REQUIRE(blocks >= 1 && blocks <= 8 && blocks <= p.k_blocks && p.M <= 256 && c.stages >= 1,
                 "gemm_int8: clusters of %d blocks do not take %d rows of %d k blocks", blocks, p.M, p.k_blocks);
    CUtensorMap map_a;
    const int rc = byte_map_for(p.a, p.M, p.K, p.lda, c.ntok, true, &map_a);
    if (rc != JLLM_OK) return rc;
    uint32_t cols = 32;
    while ((int)cols < c.ntok) cols <<= 1;
    const SwapArgs g{p.w, p.scale_w, p.scale_a, p.bias, p.has_bias, p.ldo, p.accumulate, p.M, p.N, p.k_blocks, c.ntok, c.stages, c.blocks,
                     c.share, cols, p.glu, p.error_word};
    const int tiles = (p.N + 127) / 128;
    return p.out_dtype == JLLM_F32 ? launch_swap<float>(map_a, g, c, tiles, p.out, p.stream)
                                   : launch_swap<__nv_bfloat16>(map_a, g, c, tiles, p.out, p.stream);
}

template <typename Tout, int BN>
int run_pair(const Product& p) {
    const long long packed_rows = (long long)((p.N + 127) / 128) * p.k_blocks * 128;
    JLLM_REQUIRE(packed_rows < (1LL << 31), "gemm_int8: a packed weight of %lld rows of 128 bytes is too long", packed_rows);
    CUtensorMap map_a, map_w, map_out = {};
    int rc = byte_map_for(p.a, p.M, p.K, p.lda, 128, true, &map_a);
    if (rc != JLLM_OK) return rc;
    rc = byte_map_for(p.w, packed_rows, 128, 128, BN / 2, false, &map_w);
    if (rc != JLLM_OK) return rc;
    const int bulk_out = p.out_dtype == JLLM_F32 && !p.glu && p.accumulate != EPI_RELU2 && p.ldo % 4 == 0 && ((uintptr_t)p.out % 16) == 0 && !g_plain_stores;
    if (bulk_out) {
        rc = tensor_map_out_f32(p.out, p.M, p.N, p.ldo, &map_out);
        if (rc != JLLM_OK) return rc;
    }
    int pairs = resident_pairs<Tout, BN>();
    JLLM_REQUIRE(pairs >= 1, "gemm_int8: the device runs no cluster of two blocks with %zu bytes of shared memory", PairShape<BN>::SMEM);
    const long long tiles = (long long)((p.M + 255) / 256) * ((p.N + BN - 1) / BN);
    JLLM_REQUIRE(tiles < (1LL << 31) - 1024, "gemm_int8: %lld tiles", tiles);
    if (pairs > tiles) pairs = (int)tiles;
    jllm_launch(gemm_int8_pair_kernel<Tout, BN>, dim3(2 * pairs), dim3(THREADS), PairShape<BN>::SMEM, p.stream, LAUNCH_DEPENDENT, map_a, map_w,
                map_out, bulk_out, p.scale_a, p.scale_w, p.bias, p.has_bias, (Tout*)p.out, p.ldo, p.accumulate, p.M, p.N, p.k_blocks, p.glu,
                p.error_word);
    return jllm_check_launch("gemm_int8_pair");
}

template <typename Tout>
int run_pair_width(const Product& p, int width) {
    switch (width) {
        case 256: return run_pair<Tout, 256>(p);
        case 128: return run_pair<Tout, 128>(p);
        case 64: return run_pair<Tout, 64>(p);
        default: return jllm_fail(JLLM_BAD_ARGUMENT, "gemm_int8: tiles of 64, 128 or 256 weight rows, not %d", width);
    }
}

// Blocks of a cluster (swap), or minus the tile's weight rows (pair).
int choose(int M, int N, int k_blocks, int sms) {
    const int tiles = (N + 127) / 128;
    if (M <= 256) {
        int blocks = sms / tiles;
        if (blocks > 8) blocks = 8;
        if (blocks > k_blocks) blocks = k_blocks;
        if (blocks < 1) blocks = 1;
        while (blocks > 1 && swap_cut(blocks, M, k_blocks).stages < 1) --blocks;
        return blocks;
    }
    const long long tiles_m = (M + 255) / 256, pairs = sms / 2 > 0 ? sms / 2 : 1;
    int best = 256;
    double least = 1e30;
    for (int width : {256, 128, 64}) {
        const long long rounds = (tiles_m * ((N + width - 1) / width) + pairs - 1) / pairs;
        const double cost = (double)rounds * (256 + width);
        if (cost < least) least = cost, best = width;
    }
    return -best;
}

}  // namespace

// `rows`: the int8 activations [M, K], their rows at multiples of 16 bytes; `weight`: ops.pack_int8 of the [N, K] weight, its scales filled
// up to a multiple of 128 and 16-byte aligned; out [M, N] (or [M, N / 2] with swiglu) float32 or bfloat16. `cut` (tests): blocks of a
// cluster (swap), minus the weight rows of a tile (pair), 0 as the sizes have it.
JLLM_EXPORT int jllm_gemm_int8(const Int8View* rows, const Int8View* weight, const void* bias, int bias_dtype, void* out, int out_dtype, int ldo,
                               int accumulate, int swiglu_word, int cut, cudaStream_t stream) {
    const int8_t *a = rows->data, *w_packed = weight->data;
    const float *scale_a = rows->scale, *scale_w = weight->scale;
    const int M = rows->rows, K = rows->cols, lda = rows->stride, N = weight->rows, k_blocks = weight->stride;
    const GluArgs glu = glu_args(swiglu_word, nullptr);
    JLLM_REQUIRE(M >= 0 && N >= 1 && K >= 1 && K <= MAX_K && weight->cols == K, "gemm_int8: M=%d N=%d K=%d (K from 1 to %d) against a weight of %d",
                 M, N, K, MAX_K, weight->cols);
    JLLM_REQUIRE(lda >= K && lda % 16 == 0 && ((uintptr_t)a % 16) == 0 && ((uintptr_t)w_packed % 16) == 0 && ((uintptr_t)scale_w % 16) == 0,
                 "gemm_int8: rows and weights begin at multiples of 16 bytes (lda=%d, K=%d)", lda, K);
    JLLM_REQUIRE(k_blocks == (K + BK - 1) / BK, "gemm_int8: the packed weight has %d k blocks, K=%d needs %d", k_blocks, K, (K + BK - 1) / BK);
    JLLM_REQUIRE(accumulate >= EPI_STORE && accumulate <= EPI_RELU2, "gemm_int8: accumulate=%d", accumulate);
    JLLM_REQUIRE(ldo >= (glu ? N / 2 : N), "gemm_int8: ldo=%d < N=%d", ldo, N);
    JLLM_REQUIRE(!glu || (N % 16 == 0 && !bias && !accumulate),
                 "gemm_int8: the SwiGLU epilogue needs N %% 16 == 0, no bias and no accumulation (N=%d)", N);
    if (M == 0) return JLLM_OK;
    int* error_word = jllm_gemm_error_word();
    if (!error_word) return jllm_fail(JLLM_CUDA_ERROR, "gemm_int8: no error word");
    const Product p{a, w_packed, lda, scale_a, scale_w, k_blocks, VecRef{bias, bias_dtype}, (int)(bias != nullptr), out, out_dtype, ldo, accumulate,
                    M, N, K, glu, error_word, stream};
    if (cut == 0) cut = choose(M, N, k_blocks, jllm_device_sm_count() > 0 ? jllm_device_sm_count() : 1);
    if (cut > 0) return run_swap(p, cut);
    return out_dtype == JLLM_F32 ? run_pair_width<float>(p, -cut) : run_pair_width<__nv_bfloat16>(p, -cut);
}
