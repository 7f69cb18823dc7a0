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
// The weight rows are the M side of the MMAs and the tokens the N side, so that tokens are filled up to a multiple of 16 and not of 128. A cluster of
// one to eight blocks has 128 weight rows and a group of up to 256 tokens, each block a part of the k blocks. The waits on barriers in shared
// memory end by the clock and raise the products' error word (31: the producer, 32: the MMAs, 33: the epilogue; the first one stays). Without a
// limit, as in every kernel, are the waits of the hardware itself: for the grid in front, for tensor memory, for the cluster's barrier (which
// every block reaches on every path).
#include "tcgen05_common.cuh"
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

// The result from the exact sum: the same operations in the same order for every cut.
__device__ __forceinline__ float scaled(uint32_t sum, float scale_a, float scale_w) {
    return __fmul_rn(__fmul_rn((float)(int)sum, scale_a), scale_w);
}

// What happens to the sums.
struct Finish {
    VecRef bias;
    int has_bias, ldo, accumulate, M, N;
    GluArgs glu;
};
// Results leave 16 bytes a lane: a warp parks its 32 weight rows x J tokens in shared memory and takes them back token by token. A lane
// that stores its own values stores 2 bytes of every token's row, with all that a store costs (84 ns a token and block, now 25).
template <typename Tout>
struct TokenEpilogue {
    const Finish& f;
    Tout* out;
    Tout* park;                // the warp's: 16 x 32 values, 16-byte aligned
    const float* token_scales; // shared memory, of the tokens from `first` on, 16-byte aligned
    int first, end, n, lane;   // the group's tokens [first, end); n: this lane's weight row
    float sw, b;               // its scale and its bias
    bool vec;

    __device__ __forceinline__ TokenEpilogue(const Finish& f_, Tout* out_, Tout* park_, const float* token_scales_, int n_, int lane_, float sw_)
        : f(f_), out(out_), park(park_), token_scales(token_scales_), first(0), end(0), n(n_), lane(lane_), sw(sw_),
          b(f_.has_bias && n_ < f_.N ? f_.bias[n_] : 0.f),
          vec(n_ - lane_ + 32 <= f_.N && ((uintptr_t)out_ & 15u) == 0 && (((size_t)f_.ldo * sizeof(Tout)) & 15u) == 0) {}

    // the sums of the tokens [t, t + J) for this lane's weight row; the whole warp calls it
    template <int J>
    __device__ __forceinline__ void operator()(const uint32_t (&sum)[J], int t) const {
        constexpr int PER = 16 / sizeof(Tout);       // values of a 16-byte piece
        float v[J];
#pragma unroll
        for (int j = 0; j < J; j += 4) {
            const float4 sa = *reinterpret_cast<const float4*>(token_scales + (t - first) + j);
            v[j] = scaled(sum[j], sa.x, sw);
            v[j + 1] = scaled(sum[j + 1], sa.y, sw);
            v[j + 2] = scaled(sum[j + 2], sa.z, sw);
            v[j + 3] = scaled(sum[j + 3], sa.w, sw);
        }
        const bool add_behind = sizeof(Tout) == 4 && f.accumulate == EPI_ADD;      // (a bfloat16 sum is rounded once, so it is made here)
        if (f.glu) {
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
            glu_units<J / 2, true>(f.glu.word, [&](int j) { return gate[j]; }, [&](int j) { return up[j]; }, 1.f, units);
#pragma unroll
            for (int j = 0; j < J / 2; ++j) park[(up_lane ? J / 2 + j : j) * 16 + (lane >> 4) * 8 + (lane & 7)] = from_float<Tout>(units[j]);
        } else {
            if (f.has_bias)
#pragma unroll
                for (int j = 0; j < J; ++j) v[j] = __fadd_rn(v[j], b);
            if (f.accumulate == EPI_RELU2)
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const float z = v[j] < 0.f ? 0.f : v[j];              // (what is not a number stays so: a maximum would drop it)
                    v[j] = __fmul_rn(z, z);
                }
            if (f.accumulate == EPI_ADD && !add_behind) {
                // (all the old values are requested before the first store: a load behind a store through the same pointer would wait)
                float old[J];
#pragma unroll
                for (int j = 0; j < J; ++j) old[j] = n < f.N && t + j < end ? to_float(out[(size_t)(t + j) * f.ldo + n]) : 0.f;
#pragma unroll
                for (int j = 0; j < J; ++j) v[j] = __fadd_rn(v[j], old[j]);
            }
#pragma unroll
            for (int j = 0; j < J; ++j) park[j * 32 + lane] = from_float<Tout>(v[j]);
        }
        __syncwarp();
        if (f.glu) leave<J, 16, PER>(t, (n - lane) >> 1, f.N >> 1, false);
        else leave<J, 32, PER>(t, n - lane, f.N, add_behind);
        __syncwarp();
    }

    // parked rows of WIDTH values -> out[t + j, column ...], of tokens in front of `end` and columns in front of `last` (`vec`: all are)
    template <int J, int WIDTH, int PER>
    __device__ __forceinline__ void leave(int t, int column, int last, bool add) const {
        if (vec) {
            constexpr int PIECES = WIDTH / PER, STEPS = (J * PIECES + 31) / 32;
            uint4 piece[STEPS];
            Tout* dst[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const int i = lane + 32 * s, j = i / PIECES, c = i % PIECES * PER;
                dst[s] = i < J * PIECES && t + j < end ? out + (size_t)(t + j) * f.ldo + column + c : nullptr;
                if (dst[s]) piece[s] = *reinterpret_cast<const uint4*>(park + j * WIDTH + c);
            }
            if (add) {
                float4 old[STEPS];
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
                    if (dst[s]) old[s] = *reinterpret_cast<const float4*>(dst[s]);
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    piece[s].x = __float_as_uint(__fadd_rn(__uint_as_float(piece[s].x), old[s].x));
                    piece[s].y = __float_as_uint(__fadd_rn(__uint_as_float(piece[s].y), old[s].y));
                    piece[s].z = __float_as_uint(__fadd_rn(__uint_as_float(piece[s].z), old[s].z));
                    piece[s].w = __float_as_uint(__fadd_rn(__uint_as_float(piece[s].w), old[s].w));
                }
            }
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
                if (dst[s]) *reinterpret_cast<uint4*>(dst[s]) = piece[s];
        } else {
            const int c = lane & (WIDTH - 1);
            if (column + c < last)
#pragma unroll
                for (int j = lane / WIDTH; j < J; j += 32 / WIDTH)
                    if (t + j < end) {
                        Tout* dst = out + (size_t)(t + j) * f.ldo + column + c;
                        const Tout v = park[j * WIDTH + c];
                        *dst = add ? from_float<Tout>(__fadd_rn(to_float(v), to_float(*dst))) : v;
                    }
        }
    }
};

// ---- a cluster of blocks to 128 weight rows and a group of tokens --------------------------------------------------------------
// With few tokens the product is nothing but reading W once. Block p of a cluster streams its part of the tile's k blocks (one contiguous
// 16 KB bulk copy each, requested before the kernel in front has finished: weights are nobody's output); the accumulator [128 weight
// rows x tokens] lies in its tensor memory. Of the tokens every block finishes a share: the others send their parts of it (st.async,
// which counts its bytes on the owner's mbarrier: one way through the cluster), the owner adds them up, scales and stores.
// Bound by memory where the weight is large: one row against 24,576 x 4,096 17.3 us (5.8 TB/s, 0.89 of the measured copy), 4,096 x 12,288
// 10.7 (4.7), 64 rows of it 11.1; below that by the way from launch to last store (about 3 us beside the stream: 5.5 us for the 16.8 MB of
// 4,096 x 4,096).
// With many tokens neither the tensor pipe nor what an SM takes in is full. 300 rows of 24,576 x 4,096, gated, take 40 us: the pipe is active for
// a third of it, 10 TB/s come from L2; 2,048 rows take 176 us alone (2.3 POP/s; 203 one behind the other under the power limit): 53% and
// 14 TB/s. A block has one tile, and barriers, tensor memory, the first copies and the epilogue are paid for each: with the cut held some 16 and
// 45 us of these do not depend on k. A ring of 200 KB, or two of 100 KB (two blocks an SM: the one's epilogue under the other's main loop), stands
// against the 1 to 2 us that a copy is on its way when all SMs ask. (Pairs of SMs with `cta_group::2` took 130 us for the 2,048 rows, 147 under the
// limit, and 29 for the 300. Models that ran them stopped now and then, and none of this product's waits gave up. The cause is not known, and that
// it lies in the pairs is not shown; they are gone because they could not be cleared.)
struct ClusterArgs {
    const int8_t* w;
    const float *scale_w, *scale_a;
    Finish f;
    int k_blocks, ntok, ring, blocks, share;        // ntok: the MMAs' N; share: tokens a block finishes; ring: below
    int groups, span;                               // groups of `span` tokens
    uint32_t tmem_cols;
    int* error_word;
};
// The ring's stages, and of a test of the waits (jllm_gemm_int8_starve_next) what never happens in it and its limit in us (0: WAIT_NS), in one
// word: an argument more is a line more of the arguments, and a product of few rows waits 0.1 us for it.
enum : int { STARVE_NOTHING = 0, STARVE_COPY = 1, STARVE_RELEASE = 2, STARVE_PARTS = 3 };
constexpr int ring_word(int stages, int starve, int limit_us) { return stages | starve << 8 | limit_us << 10; }
constexpr int MOST_LIMIT_US = 1000000;
static_assert(ring_word(255, STARVE_PARTS, MOST_LIMIT_US) > 0, "20 bits of a limit");

__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned long long limit) {
    unsigned long long began = 0;
    for (uint32_t i = 0;; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) return true;
        if ((i & 63u) == 63u) {
            const unsigned long long now = now_ns();
            if (began == 0) began = now;
            if (*abort_flag || now - began > limit) return false;
        }
    }
}
// (the bytes alone, no arrival)
__device__ __forceinline__ void mbar_expect_more(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// What is still on its way when a wait has run out: waited for whatever the others do, until `limit` after `began`.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity, unsigned long long began, unsigned long long limit) {
    while (!mbar_try_wait(bar, parity) && now_ns() - began < limit) {}
}

// (128 registers a thread: registers are dealt out for eight warps where there are six, and with more no second block fits beside one)
template <typename Tout>
__global__ void __launch_bounds__(256, 2)
gemm_int8_cluster_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ ClusterArgs g, Tout* __restrict__ out) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(16) float token_scales[256];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* aligned = smem_raw + (base - smem_u32(smem_raw));
    const int stages = g.ring & 255, starve = g.ring >> 8 & 3, blocks = g.blocks, share = g.share;
    const unsigned long long limit = g.ring >> 10 ? (g.ring >> 10) * 1000ull : WAIT_NS;
    const uint32_t stage_bytes = TILE_BYTES + (uint32_t)g.ntok * BK, parts_at = (uint32_t)stages * stage_bytes;
    const uint32_t part_bytes = (uint32_t)share * 128 * 4;         // one block's part of a share, [share / 4][128 rows][4 tokens]
    const uint32_t bars_at = parts_at + (uint32_t)(blocks - 1) * part_bytes, bars = base + bars_at;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (stages + s); };
    const uint32_t acc_bar = bars + 16u * stages, parts_bar = acc_bar + 8u;
    uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(aligned + bars_at + 8 * (2 * stages + 2));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);
    // Who waits for another role of the block waits twice as long as that one does for its copies, so that the code names what is missing.
    auto give_up = [&](int code) {
        atomicCAS(g.error_word, 0, code);
        __threadfence();               // (before anybody follows the flag and has a code of his own)
        *abort_flag = 1;
    };

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    // a cluster's 128 weight rows and its group of tokens, the groups fastest: what runs together shares its weights
    const int unit = (int)blockIdx.x / blocks, rank = (int)blockIdx.x % blocks;      // (clusters lie along x: this is the rank)
    const int tile = unit / g.groups, first = unit % g.groups * g.span, here = min(g.span, g.f.M - first);
    const int kb_lo = (int)((long long)g.k_blocks * rank / blocks), n_kb = (int)((long long)g.k_blocks * (rank + 1) / blocks) - kb_lo;
    const int tokens = (here + 7) & ~7;                               // the accumulator's columns that anybody needs
    const int mine = rank * share, mine_end = min(mine + share, tokens);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(acc_bar, 1);
        mbar_init(parts_bar, 1);
        *abort_flag = 0;
        if (starve != STARVE_NOTHING) {
            if (starve == STARVE_RELEASE) {
                asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(empty_bar(0)) : "memory");
                mbar_init(empty_bar(0), 2);
            } else if (starve == STARVE_PARTS) mbar_expect_more(parts_bar, 16);
            else if (rank == 0) mbar_expect_more(full_bar(0), 16);
        }
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
    int issued = 0;                            // k blocks whose copies (warp 0), or whose MMAs (warp 1), are under way or done
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
                tma_load_2d(base + (uint32_t)i * stage_bytes + TILE_BYTES, &map_a, (kb_lo + i) * BK, first, full_bar(i));
        __syncwarp();
        int s = 0, i = early;
        uint32_t parity = 0;                                   // the ring's second lap waits for the first lap's release
        for (; i < n_kb; ++i) {
            if (!warp_wait(empty_bar(s), parity, abort_flag, 2 * limit)) { ok = false; break; }
            if (elect_one()) {
                const uint32_t dst = base + (uint32_t)s * stage_bytes;
                mbar_expect_tx(full_bar(s), stage_bytes);
                bulk_copy(dst, w + (size_t)i * TILE_BYTES, TILE_BYTES, full_bar(s));
                tma_load_2d(dst + TILE_BYTES, &map_a, (kb_lo + i) * BK, first, full_bar(s));
            }
            __syncwarp();
            if (++s == stages) { s = 0; parity ^= 1u; }
        }
        // (the last lap's releases have arrived too before the block may leave: none is on its way to memory that is somebody else's by then)
        for (int j = max(0, n_kb - stages); ok && j < n_kb; ++j)
            ok = warp_wait(empty_bar(j % stages), (uint32_t)(j / stages) & 1u, abort_flag, 2 * limit);
        issued = i;
        if (!ok && lane == 0) give_up(31);
        if (blocks > 1) cluster_wait();
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        const uint32_t idesc = idesc_i8(128, g.ntok);
        const uint64_t desc_w0 = smem_desc_sw128(base), desc_b0 = smem_desc_sw128(base + TILE_BYTES);
        uint64_t desc_w = desc_w0, desc_b = desc_b0;          // (a stage further is an addition to the address field)
        int s = 0, i = 0;
        uint32_t parity = 0;
        pdl_wait();          // (the copies are complete no sooner, and the time that the kernel in front still takes is not this wait's)
        for (; i < n_kb; ++i) {
            if (!warp_wait(full_bar(s), parity, abort_flag, limit)) { ok = false; break; }
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
        if (ok && elect_one()) tcgen05_commit(acc_bar);
        __syncwarp();
        issued = i;
        if (!ok && lane == 0) give_up(32);
        if (blocks > 1) cluster_wait();
    } else {
        // ---------------- epilogue: warps 2..5, TMEM lanes 32 * (warp % 4) = weight rows of the tile ----------------
        const int quad = warp & 3, row = quad * 32 + lane, n = tile * 128 + row;
        const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16);
        const float sw = g.scale_w[n];                        // (filled up to whole tiles)
        // (parks in the ring, which is idle once every MMA is done)
        TokenEpilogue<Tout> finish(g.f, out, reinterpret_cast<Tout*>(aligned + (size_t)quad * 2048), token_scales, n, lane, sw);
        finish.first = first;
        finish.end = first + here;
        pdl_wait();          // the token scales, and what is added into, were written by the kernels before
        pdl_trigger();
        // (into shared memory while the weights come: asked for in front of every store they were 1 us for 8 tokens)
        for (int i = threadIdx.x - 64; i < 256; i += 128) token_scales[i] = i < here ? g.scale_a[first + i] : 0.f;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (blocks > 1) cluster_wait();
        ok = mbar_wait(acc_bar, 0, abort_flag, 2 * limit);
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
        if (ok && blocks > 1 && mine < mine_end) ok = __all_sync(0xffffffffu, wait_cluster(parts_bar, 0, abort_flag, 2 * limit));
        if (ok) {
            const uint8_t* parts = aligned + parts_at + (size_t)row * 16;
            auto add_up = [&](auto& sum, int t) {
                tmem_ld(taddr + t, sum);
                tmem_ld_wait();
                for (int p = 0; p < blocks - 1; ++p) {
                    const uint8_t* src = parts + (size_t)p * part_bytes + (size_t)((t - mine) / 4) * 2048;
#pragma unroll
                    for (int q = 0; q < (int)(sizeof(sum) / 16); ++q) {
                        const uint4 x = *reinterpret_cast<const uint4*>(src + q * 2048);
                        sum[4 * q] += x.x, sum[4 * q + 1] += x.y, sum[4 * q + 2] += x.z, sum[4 * q + 3] += x.w;
                    }
                }
                finish(sum, first + t);
            };
            int t = mine;
            uint32_t sum16[16], sum8[8];
#pragma unroll 1
            for (; t + 16 <= mine_end; t += 16) add_up(sum16, t);
            if (t < mine_end) add_up(sum8, t);
        } else if (lane == 0) give_up(33);
    }
    tcgen05_fence_before();
    const bool gave_up = __syncthreads_or(!ok);
    if (gave_up) {
        // (where no wait ran out these have been waited for: the copies by the MMAs, the MMAs by the epilogue and the producer)
        const unsigned long long began = now_ns();
        if (warp == 0)
            for (int j = max(0, issued - stages); j < issued; ++j) drain(full_bar(j % stages), (uint32_t)(j / stages) & 1u, began, limit);
        if (warp == 1 && issued > 0) drain(empty_bar((issued - 1) % stages), (uint32_t)((issued - 1) / stages) & 1u, began, limit);
        __syncthreads();
    }
    if (warp == 2) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(g.tmem_cols) : "memory");
    }
    // No block leaves before everything sent to it is there: its memory is the next block's at once. A block whose epilogue went through has
    // waited for its parts; one that gave up, or whose neighbours did, waits for them here, behind the barrier that all sends are made in front
    // of, for as long as a wait may last (parts that were never sent do not come; one that was sent takes microseconds).
    if (blocks > 1) {
        cluster_arrive();
        cluster_wait();
        if (gave_up) drain(parts_bar, 0, now_ns(), limit);
    }
}

struct ClusterCut {
    int blocks, share, ntok, stages, groups, span;
    size_t smem;
};
// `deep`: the ring takes all shared memory of an SM, else half of it, so that a second block (of this product, or of the next one, whose first
// weights then come while this one ends) fits beside.
ClusterCut cluster_cut(int blocks, bool deep, int groups, int M, int k_blocks) {
    const int span = (int)((((long long)M + groups - 1) / groups + 15) / 16 * 16);          // (the last group may be short, or there are fewer)
    ClusterCut c{blocks, (span / 8 + blocks - 1) / blocks * 8, span, 0, (M + span - 1) / span, span, 0};
    if (span > 256) return c;
    if (groups == 1) c.share = ((M + 7) / 8 + blocks - 1) / blocks * 8;
    const size_t stage = TILE_BYTES + (size_t)c.ntok * BK, parts = (size_t)(blocks - 1) * c.share * 512;
    const size_t room = deep ? SMEM_ROOM - 4096 : 104 * 1024;
    c.stages = parts + 2 * stage > room ? 0 : (int)((room - parts) / stage);
    const int most = (k_blocks + blocks - 1) / blocks;
    if (c.stages > most) c.stages = most;
    c.smem = c.stages * stage + parts + 1024 + 8 * (2 * c.stages + 2) + 16;
    // Blocks that wait for one another must not wait for tensor memory that others hold who wait in turn: the blocks on an SM never ask for
    // more than its 512 columns. Of 60 KB and more (less 128 columns each) there are at most three, of 114 KB one beside another; a block that
    // takes all columns (of this file or another) has over 190 KB.
    const size_t least = blocks == 1 ? 0 : c.ntok > 128 ? 114 * 1024 : 60 * 1024;
    if (c.smem < least) c.smem = least;
    return c;
}

// ---- host side ----------------------------------------------------------------------------------------------------------

// A [rows, cols] matrix of bytes with row stride ld, read in boxes of box_rows x 128 with the 128-byte swizzle.
int byte_map_for(const void* ptr, long long rows, long long cols, long long ld, int box_rows, CUtensorMap* out) {
    static std::unordered_map<MapKey, CUtensorMap, MapKeyHash> cache;
    static std::mutex mu;
    const MapKey key{ptr, rows, cols, ld, box_rows};
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
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return jllm_fail(JLLM_CUDA_ERROR, "gemm_int8: cuTensorMapEncodeTiled failed (%d) for [%lld, %lld] bytes, ld %lld", (int)r, rows, cols, ld);
    if (cache.size() > 4096) cache.clear();
    cache.emplace(key, map);
    *out = map;
    return JLLM_OK;
}

cudaLaunchConfig_t cluster_config(const ClusterCut& c, int tiles, cudaLaunchAttribute* attr, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * c.blocks);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = c.smem;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c.blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cfg;
}

template <typename Tout>
int launch_cluster(const CUtensorMap& map_a, const ClusterArgs& g, const ClusterCut& c, int tiles, void* out, cudaStream_t stream) {
    auto kern = gemm_int8_cluster_kernel<Tout>;
    if (jllm_allow_smem((const void*)kern, c.smem) != cudaSuccess)
        return jllm_fail(JLLM_CUDA_ERROR, "gemm_int8: %zu bytes of shared memory refused", c.smem);
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = cluster_config(c, tiles, attr, stream);
    if (jllm_launch_overlaps(c.smem, LAUNCH_DEPENDENT)) {
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 2;
    }
    cudaLaunchKernelEx(&cfg, kern, map_a, g, static_cast<Tout*>(out));
    return jllm_check_launch("gemm_int8_cluster");
}

// clusters of that many blocks that the device runs at a time, one block an SM; asked once per device
template <typename Tout>
int resident_clusters(int blocks) {
    static int known[64][9] = {};          // (one more than the answer)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (known[dev][blocks]) return known[dev][blocks] - 1;
    int n = 0;
    ClusterCut one{};
    one.blocks = blocks, one.smem = SMEM_ROOM;
    cudaLaunchAttribute attr[1];
    const cudaLaunchConfig_t cfg = cluster_config(one, 1, attr, nullptr);
    if (jllm_allow_smem((const void*)gemm_int8_cluster_kernel<Tout>, SMEM_ROOM) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, gemm_int8_cluster_kernel<Tout>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    known[dev][blocks] = n + 1;
    return n;
}

// A test of the waits: what the next product of this thread is to miss, and how long its waits last.
struct Starve {
    int what, limit_us;
};
thread_local Starve g_starve_next = {STARVE_NOTHING, 0};

struct Product {
    const int8_t *a, *w;
    int lda;
    const float *scale_a, *scale_w;
    int k_blocks, K;
    void* out;
    int out_dtype;
    Finish f;
    int* error_word;
    cudaStream_t stream;
    Starve starve;
};

// What stands for a cut in one number: the blocks of a cluster, 10 more with a deep ring, 100 more for each group of tokens
constexpr int DEEP = 10, GROUP = 100;
struct Cut {
    int blocks, groups;
    bool deep;
};
Cut cut_of(int code, int M) {
    const int groups = code / GROUP;
    return {code % DEEP, groups > 0 ? groups : (M + 255) / 256, code % GROUP > DEEP};
}

int run_cluster(const Product& p, int code) {
    const int M = p.f.M;
    const Cut cut = cut_of(code, M);
    JLLM_REQUIRE(code > 0 && code % GROUP < 2 * DEEP && cut.blocks >= 1 && cut.blocks <= 8 && cut.blocks <= p.k_blocks && cut.groups <= M,
                 "gemm_int8: no cut %d for %d rows of %d k blocks", code, M, p.k_blocks);
    const ClusterCut c = cluster_cut(cut.blocks, cut.deep, cut.groups, M, p.k_blocks);
    JLLM_REQUIRE(c.stages >= 1, "gemm_int8: clusters of %d blocks do not take %d rows in %d groups", cut.blocks, M, cut.groups);
    const long long units = (long long)((p.f.N + 127) / 128) * c.groups;
    JLLM_REQUIRE(units * c.blocks < (1LL << 31) && (long long)(c.groups + 1) * c.span < (1LL << 31), "gemm_int8: %lld tiles of %d rows", units, M);
    JLLM_REQUIRE(p.starve.what == STARVE_NOTHING || (units * c.blocks <= 64 && (p.starve.what != STARVE_PARTS || c.blocks > 1)),
                 "gemm_int8: the starved product of the wait test has at most 64 blocks, and a cluster where parts are missed");
    CUtensorMap map_a;
    const int rc = byte_map_for(p.a, M, p.K, p.lda, c.ntok, &map_a);
    if (rc != JLLM_OK) return rc;
    uint32_t cols = 32;
    while ((int)cols < c.ntok) cols <<= 1;
    const ClusterArgs g{p.w, p.scale_w, p.scale_a, p.f, p.k_blocks, c.ntok, ring_word(c.stages, p.starve.what, p.starve.limit_us), c.blocks, c.share,
                        c.groups, c.span, cols, p.error_word};
    return p.out_dtype == JLLM_F32 ? launch_cluster<float>(map_a, g, c, (int)units, p.out, p.stream)
                                   : launch_cluster<__nv_bfloat16>(map_a, g, c, (int)units, p.out, p.stream);
}

// A count that puts the cuts in order. Its terms follow what a product does and its constants are fitted so that the least count is a fast cut, to
// products launched back to back on weights larger than L2; a constant is no duration and a count no time (300 plain rows of 24,576 x 4,096
// count 28 and take 37 us, 2,048 count 133 and take 174).
// Up to 256 rows (one group; 846 sizes of 1 to 256 rows against 128 to 34,816 weight rows of 256 to 17,408 values: what is chosen is 2.1% slower than
// the best way of each size in the geometric mean): a block's k blocks, each 1.13 shared by the ring's stages (a copy's way) or 0.12 and 0.00055 a
// token (the MMAs); all clusters at once, one block an SM, or (half of that a round) two blocks side by side, or one batch behind the other; 0.3 where
// nothing of the next product lies beside it; sending 0.15 a block of the cluster and 0.01 a token sent; the weights' bytes by READ_BYTES_US at least.
constexpr double READ_BYTES_US = 1e7;
template <typename Tout>
double cluster_cost(int M, int N, int k_blocks, const Cut& cut) {
    const ClusterCut c = cluster_cut(cut.blocks, cut.deep, cut.groups, M, k_blocks);
    if (cut.blocks > k_blocks || c.stages < 1) return 1e30;
    // (the driver counts one block an SM for whatever allocates tensor memory; two run where shared memory has room)
    const long long units = (long long)((N + 127) / 128) * c.groups;
    const int alone = resident_clusters<Tout>(cut.blocks), beside = c.smem + 2048 <= 114 * 1024 ? 2 * alone : alone;
    if (alone < 1) return 1e30;
    const double flow = 0.12 + 0.00055 * c.ntok, lag = 1.13 / c.stages;
    const double each = (double)((k_blocks + cut.blocks - 1) / cut.blocks) * (flow > lag ? flow : lag);
    const double waves = (double)((units + alone - 1) / alone), batches = (double)((units + beside - 1) / beside);
    const double run = beside == alone ? waves * (each + 1.2) - 1.2 + 0.3 : (waves > 1 ? 0.5 * waves : 1.0) * each + (batches - 1) * 1.2;
    const double read = (double)N * k_blocks * BK / READ_BYTES_US;
    return (run > read ? run : read) + (cut.blocks > 1 ? 0.15 * cut.blocks + 0.01 * (c.ntok - c.share) : 0.0) + 0.007 * (c.share < c.ntok ? c.share : c.ntok);
}

// More rows (groups of them; 162 sizes of 300 to 2,048 rows against 1,024 to 24,576 weight rows of 1,024 to 12,288 values: 1.6%): all SMs take in at once.
// One block an SM: rounds of k blocks, each 1.06 shared by the stages or 0.135 and 0.00027 a token, and 1.9 and 0.0104 a token to begin and end. Two
// blocks side by side: the SM's share of all k blocks at 0.215 and 0.00025 a token (or 1.45 shared by both rings), an end that shows once, 2 a batch.
// Sending 0.55 a block of the cluster and 0.043 a token.
template <typename Tout>
double groups_cost(int M, int N, int k_blocks, const Cut& cut) {
    const ClusterCut c = cluster_cut(cut.blocks, cut.deep, cut.groups, M, k_blocks);
    if (cut.blocks > k_blocks || c.stages < 1) return 1e30;
    const long long units = (long long)((N + 127) / 128) * c.groups;
    const int alone = resident_clusters<Tout>(cut.blocks), sms = resident_clusters<Tout>(1), beside = c.smem + 2048 <= 114 * 1024 ? 2 * alone : alone;
    if (alone < 1 || sms < 1) return 1e30;
    const int each_kb = (k_blocks + cut.blocks - 1) / cut.blocks, mine = c.share < c.ntok ? c.share : c.ntok;
    const double flow = 0.135 + 0.00027 * c.ntok, lag = 1.06 / c.stages, each = each_kb * (flow > lag ? flow : lag), end = 0.0104 * mine;
    const double waves = (double)((units + alone - 1) / alone), batches = (double)((units + beside - 1) / beside);
    double run = waves * (each + 1.9 + end);
    if (beside > alone) {
        const double two = 0.215 + 0.00025 * c.ntok, two_lag = 1.45 / (2 * c.stages);
        run = each + end;
        if (waves > 1) {
            const double shared = (double)(units * cut.blocks) / sms * each_kb * (two > two_lag ? two : two_lag);
            run = (run > shared ? run : shared) + end;
        }
        run += (batches - 1) * 2.0;
    }
    return run + (cut.blocks > 1 ? 0.55 * cut.blocks + 0.043 * (c.ntok - c.share) : 0.0);
}

// The cut for a product. (Worked out once per size: the choice is kept.)
template <typename Tout>
int choose(int M, int N, int k_blocks) {
    static std::mutex mu;
    static std::unordered_map<MapKey, int, MapKeyHash> known;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    const MapKey key{nullptr, M, N, k_blocks, dev};
    std::lock_guard<std::mutex> lock(mu);
    const auto it = known.find(key);
    if (it != known.end()) return it->second;
    int best = 1 + GROUP * ((M + 255) / 256);
    double least = 1e30;
    for (int span = 16; span <= 256; span += 16) {
        if (M <= 256 && span < (M + 15) / 16 * 16) continue;         // (few tokens are one group: another would read the weights again)
        const int groups = (M + span - 1) / span;
        for (int ring = 0; ring < 2; ++ring)
            for (int blocks = 1; blocks <= 8; ++blocks) {
                const Cut cut{blocks, groups, ring == 1};
                const double cost = M <= 256 ? cluster_cost<Tout>(M, N, k_blocks, cut) : groups_cost<Tout>(M, N, k_blocks, cut);
                if (cost < least) least = cost, best = blocks + DEEP * ring + GROUP * groups;
            }
        if (M <= 256) break;
    }
    if (known.size() >= 4096) known.clear();
    return known[key] = best;
}

}  // namespace

int* jllm_gemm_error_word();

// A test of the bounded waits: the NEXT product of this thread has waits of `limit_us` microseconds, and with `what` 1 a copy's barrier that
// expects more than comes, with 2 a stage that is never released, with 3 a part that no block of the cluster sends (0: the limit alone). It
// returns, raises the error word and leaves the device usable.
JLLM_EXPORT int jllm_gemm_int8_starve_next(int what, int limit_us) {
    JLLM_REQUIRE(what >= STARVE_NOTHING && what <= STARVE_PARTS && limit_us >= 1 && limit_us <= MOST_LIMIT_US, "gemm_int8_starve_next: %d, %d us", what, limit_us);
    g_starve_next = {what, limit_us};
    return JLLM_OK;
}

// `rows`: the int8 activations [M, K], their rows at multiples of 16 bytes; `weight`: ops.pack_int8 of the [N, K] weight, its scales filled
// up to a multiple of 128 and 16-byte aligned; out [M, N] (or [M, N / 2] with swiglu) float32 or bfloat16. `cut` (tests): blocks of a
// cluster, 10 more with a ring of all of an SM's shared memory, 100 more for each group of tokens; 0 as the sizes have it.
JLLM_EXPORT int jllm_gemm_int8(const Int8View* rows, const Int8View* weight, const void* bias, int bias_dtype, void* out, int out_dtype, int ldo,
                               int accumulate, int swiglu_word, int cut, cudaStream_t stream) {
    const int8_t *a = rows->data, *w_packed = weight->data;
    const float *scale_a = rows->scale, *scale_w = weight->scale;
    const int M = rows->rows, K = rows->cols, lda = rows->stride, N = weight->rows, k_blocks = weight->stride;
    const GluArgs glu = glu_args(swiglu_word, nullptr);
    const Starve starve = g_starve_next;
    g_starve_next = {STARVE_NOTHING, 0};
    JLLM_REQUIRE(M >= 0 && M <= INT8_MOST && N >= 1 && K >= 1 && K <= MAX_K && weight->cols == K, "gemm_int8: M=%d N=%d K=%d (K from 1 to %d) against a weight of %d",
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
    const Product p{a, w_packed, lda, scale_a, scale_w, k_blocks, K, out, out_dtype,
                    Finish{VecRef{bias, bias_dtype}, (int)(bias != nullptr), ldo, accumulate, M, N, glu}, error_word, stream, starve};
    if (cut == 0) cut = out_dtype == JLLM_F32 ? choose<float>(M, N, k_blocks) : choose<__nv_bfloat16>(M, N, k_blocks);
    return run_cluster(p, cut);
}
