// Products of ragged groups of rows, each with a weight of its own, and products in 8-bit floating point, on the 5th-generation tensor cores:
//
//   out[p, n] = sum_k a[row(p), k] * w[g(p), n, k]                                                        (bfloat16)
//   out[p, n] = sum_b scale_a[row(p), b] * scale_w[g(p), n / 128, b] * sum_(k in block b) qa[row(p), k] * qw[g(p), n, k]      (e4m3, b: 128 k)
//
// The pairs p of a group g are neighbours (offsets[g] .. offsets[g + 1]); a pair's row is the pair itself, or the token that asked (order[p] /
// top), whose row is then fetched where it lies: nothing is copied together first. A product of rows with one weight is the case of one group.
//
// The weight is PACKED once: tiles of 128 rows x 128 bytes of k (64 bfloat16, 128 e4m3), each the 16 KB image that the tensor cores read from
// shared memory (16-byte chunk c of row r at chunk position c ^ (r & 7)), tile t of group g at k block kb at ((g * tiles + t) * k_blocks + kb) *
// 16 KB. The weight rows are the M side of the MMAs and the rows of a group the N side, filled up to a multiple of 16: of the many small groups of
// a step nothing is wasted on a side of 128. A unit of work is MT tiles of a group's weight and a span of up to NT of its pairs.
//
// The blocks stay: block b takes the units b, b + blocks, ... of a list that every block reckons by itself from the offsets (the host does not
// know them). Warp 0 brings tiles (bulk copies of weights, TMA boxes or gathers of four rows of activations) into a ring that runs on over the
// units, warp 1 issues the MMAs, the others take the sums from tensor memory. So the copies of the next unit are under way while this one ends.
//
// In 8 bits the sums of ONE k block are made by the tensor cores (float32) and lie in one of several buffers in tensor memory; the epilogue warps
// multiply them by both scales and add them into float32 registers. The scales of a block are float32 numbers of any value: the hardware's own
// block scales are powers of two for 32 values each.
//
// A product of few rows whose tiles do not fill the SMs: `blocks` blocks of a cluster share a unit's k blocks and send their parts (st.async)
// to the block that finishes the token; parts are added in a fixed order.
//
// The waits on barriers in shared memory end by the clock and raise the products' error word (41: the producer, 42: the MMAs, 43: the epilogue).
#include "fp8_view.h"
#include "tcgen05_common.cuh"

namespace {

using namespace tc;

constexpr int TILE_BYTES = 128 * 128;
constexpr int MAX_GROUPS = 1024;

struct Finish {
    VecRef bias;
    int has_bias, ldo, accumulate, N, glu;
};

struct Args {
    const uint8_t* w;
    const float *scale_w, *scale_a;       // [groups, tiles * 16, sw_ld] and [rows, sa_ld]: multiples of four values a row
    const int *offsets, *order;           // null: one group of `rows`; null: a pair's row is the pair
    int sw_ld, sa_ld;
    int groups, top, rows, tiles, k_blocks;
    Finish f;
    int stages, blocks, share;            // blocks of a cluster, tokens that each of them finishes
    int starve, limit_us;                 // a test of the waits (below); 0, 0
    int* error_word;
};
enum : int { STARVE_NOTHING = 0, STARVE_COPY = 1, STARVE_RELEASE = 2, STARVE_PARTS = 3 };

// A unit: tiles [tile, tile + MT) of group e's weight against `here` pairs from `first` on, filled up to `width`.
struct Unit {
    int e, tile, first, here, width;
};

// kind::f16 (bfloat16) and kind::f8f6f4 (e4m3): float32 accumulators, both operands K-major
template <bool FP8>
__device__ __forceinline__ uint32_t idesc(int n) {
    return (1u << 4) | (FP8 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
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
// Four rows of a matrix (each with a row number of its own), one under the other: the tensor map's box is one row high.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int x, const int (&row)[4], uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(map), "r"(x), "r"(row[0]), "r"(row[1]), "r"(row[2]), "r"(row[3]), "r"(bar)
        : "memory");
}
__device__ __forceinline__ uint64_t pair_of(uint32_t a, uint32_t b) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "r"(a), "r"(b));
    return p;
}
__device__ __forceinline__ void halves(uint64_t p, float& a, float& b) {
    uint32_t x, y;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(x), "=r"(y) : "l"(p));
    a = __uint_as_float(x), b = __uint_as_float(y);
}
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

// Units in front of every group, by the whole block (a lane has 32 neighbouring groups at most); a __syncthreads has to follow.
template <int NT, int MT>
__device__ __forceinline__ void list_units(const Args& g, int* before, int* at) {
    pdl_wait();          // (the offsets are the kernel in front's)
    for (int i = threadIdx.x; i <= g.groups; i += blockDim.x) at[i] = g.offsets[i];
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x, each = (g.groups + 31) / 32, lo = min(lane * each, g.groups), hi = min(lo + each, g.groups), tiles = (g.tiles + MT - 1) / MT;
    int sum = 0;
    for (int i = lo; i < hi; ++i) sum += (at[i + 1] - at[i] + NT - 1) / NT * tiles;
    int run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int left = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += left;
    }
    run -= sum;
    for (int i = lo; i < hi; ++i) {
        before[i] = run;
        run += (at[i + 1] - at[i] + NT - 1) / NT * tiles;
    }
    if (lane == 31) before[g.groups] = run;
}

// The list of units, in the order that the blocks walk it: groups, of a group the tiles, of a tile the spans (which share its weights).
// `before`: shared memory, units in front of every group; `at`: where its pairs begin. Without offsets there is one group of `rows`.
template <int NT, int MT>
struct Units {
    const Args& g;
    const int *before, *at;
    int total, tiles;
    int e = 0;                            // the group of the unit that was asked for last (units are asked for in ascending order)

    __device__ __forceinline__ Units(const Args& g_, const int* before_, const int* at_) : g(g_), before(before_), at(at_), tiles((g_.tiles + MT - 1) / MT) {
        total = g.offsets ? before[g.groups] : tiles * ((g.rows + NT - 1) / NT);
    }
    // the whole warp calls it
    __device__ __forceinline__ Unit operator()(int u) {
        int count = g.rows, first = 0, r = u;
        if (g.offsets) {
            const int lane = threadIdx.x & 31;
            for (;;) {                    // (before[groups] = total > u: it ends)
                const int i = e + 1 + lane;
                const unsigned behind = __ballot_sync(0xffffffffu, i <= g.groups && before[i] <= u);
                e += __popc(behind);
                if (behind != 0xffffffffu) break;
            }
            first = at[e], count = at[e + 1] - first, r = u - before[e];
        }
        const int spans = (count + NT - 1) / NT, width = ((count + spans - 1) / spans + 15) & ~15, s = r % spans;
        return {e, r / spans * MT, first + s * width, min(width, count - s * width), width};
    }
};

// 16 pairs x 32 weight rows of a warp, parked in shared memory as [16][32] floats -> out, pairs [lo, hi) of the 16 that begin at row p0,
// 16 bytes a lane where `vec`.
template <typename Tout>
__device__ __forceinline__ void leave(const Finish& f, Tout* out, const float* park, size_t p0, int lo, int hi, int n0, bool vec, int lane) {
    constexpr int PER = 16 / sizeof(Tout);
    if (f.glu) {
        // rows come in blocks of 16: 8 gate rows and the 8 up rows of the same hidden units
        const int u0 = n0 >> 1, last = f.N >> 1;
        if (vec) {
#pragma unroll
            for (int i = lane; i < 16 * (16 / PER); i += 32) {
                const int j = i / (16 / PER), c = i % (16 / PER) * PER;
                if (j < lo || j >= hi) continue;
                const float* src = park + j * 32 + (c >> 3) * 16 + (c & 7);
                float gate[PER], up[PER], units[PER];
#pragma unroll
                for (int q = 0; q < PER; q += 4) {
                    *reinterpret_cast<float4*>(gate + q) = *reinterpret_cast<const float4*>(src + q);
                    *reinterpret_cast<float4*>(up + q) = *reinterpret_cast<const float4*>(src + 8 + q);
                }
                glu_units<PER, true>(f.glu, [&](int q) { return gate[q]; }, [&](int q) { return up[q]; }, 1.f, units);
                __align__(16) Tout v[PER];
#pragma unroll
                for (int q = 0; q < PER; ++q) v[q] = from_float<Tout>(units[q]);
                *reinterpret_cast<uint4*>(out + (p0 + j) * f.ldo + u0 + c) = *reinterpret_cast<const uint4*>(v);
            }
        } else {
            const int c = lane & 15;
            for (int j = lo + (lane >> 4); j < hi; j += 2) {
                const float* src = park + j * 32 + (c >> 3) * 16 + (c & 7);
                const float gate = src[0], up = src[8];
                float units[1];
                glu_units<1, true>(f.glu, [&](int) { return gate; }, [&](int) { return up; }, 1.f, units);
                if (u0 + c < last) out[(p0 + j) * f.ldo + u0 + c] = from_float<Tout>(units[0]);
            }
        }
        return;
    }
    if (vec) {
#pragma unroll
        for (int i = lane; i < 16 * (32 / PER); i += 32) {
            const int j = i / (32 / PER), c = i % (32 / PER) * PER;
            if (j < lo || j >= hi) continue;
            Tout* dst = out + (p0 + j) * f.ldo + n0 + c;
            float v[PER];
#pragma unroll
            for (int q = 0; q < PER; q += 4) *reinterpret_cast<float4*>(v + q) = *reinterpret_cast<const float4*>(park + j * 32 + c + q);
            __align__(16) Tout w[PER];
            if (f.accumulate == EPI_ADD) {
                *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(dst);
#pragma unroll
                for (int q = 0; q < PER; ++q) v[q] = __fadd_rn(v[q], to_float(w[q]));
            }
#pragma unroll
            for (int q = 0; q < PER; ++q) w[q] = from_float<Tout>(v[q]);
            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(w);
        }
    } else if (n0 + lane < f.N) {
        for (int j = lo; j < hi; ++j) {
            Tout* dst = out + (p0 + j) * f.ldo + n0 + lane;
            const float v = park[j * 32 + lane];
            *dst = from_float<Tout>(f.accumulate == EPI_ADD ? __fadd_rn(v, to_float(*dst)) : v);
        }
    }
}

// What a variant takes of an SM: buffers of accumulators in tensor memory, threads.
template <bool FP8, int NT, int MT>
struct Shape {
    // (in 8 bits a buffer is one k block's sums, else a unit's)
    static constexpr int BUFFERS = !FP8 ? 2 : MT * NT * 4 <= 256 ? 4 : 2;
    static constexpr int COLUMNS = BUFFERS * MT * NT < 32 ? 32 : BUFFERS * MT * NT;
    static constexpr int EPILOGUE = 4 * MT, THREADS = 64 + 32 * EPILOGUE;
    static constexpr uint32_t STAGE = MT * TILE_BYTES + NT * 128;
    static_assert(COLUMNS <= 512 && (COLUMNS & (COLUMNS - 1)) == 0, "tensor memory is dealt out in powers of two");
};

template <bool FP8, int NT, int MT, typename Tout>
__global__ void __launch_bounds__(64 + 128 * MT, NT <= 64 ? 2 : 1)
gemm_grouped_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ Args g, Tout* __restrict__ out) {
    using S = Shape<FP8, NT, MT>;
    constexpr int CHUNKS = NT / 16;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int before[MAX_GROUPS + 1], at[MAX_GROUPS + 1];
    __shared__ __align__(16) float parks[S::EPILOGUE][16 * 32];
    __shared__ __align__(16) float token_scales[FP8 ? 2 : 1][FP8 ? 4 : 1][FP8 ? NT : 4];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_word;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* aligned = smem_raw + (base - smem_u32(smem_raw));
    const int stages = g.stages, blocks = g.blocks;
    const unsigned long long limit = g.limit_us ? g.limit_us * 1000ull : WAIT_NS;
    const uint32_t parts_at = (uint32_t)stages * S::STAGE, part_bytes = (uint32_t)g.share * 128 * 4;      // [share / 4][128 rows][4 tokens]
    const uint32_t bars = base + parts_at + (uint32_t)(blocks - 1) * part_bytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (stages + s); };
    auto sums_bar = [&](int b) { return bars + 16u * stages + 8u * b; };                     // a buffer's sums are there
    auto taken_bar = [&](int b) { return bars + 16u * stages + 8u * (S::BUFFERS + b); };      // ... have been read
    const uint32_t parts_bar = bars + 16u * stages + 16u * S::BUFFERS;
    volatile int* abort_flag = &abort_word;
    // Who waits for another role of the block waits twice as long as that one does for its copies, so that the code names what is missing.
    auto give_up = [&](int code) {
        atomicCAS(g.error_word, 0, code);
        __threadfence();               // (before anybody follows the flag and has a code of his own)
        *abort_flag = 1;
    };

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int cluster = (int)blockIdx.x / blocks, clusters = (int)gridDim.x / blocks, rank = (int)blockIdx.x % blocks;
    const int kb_lo = (int)((long long)g.k_blocks * rank / blocks), n_kb = (int)((long long)g.k_blocks * (rank + 1) / blocks) - kb_lo;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1 + (g.starve == STARVE_RELEASE && s == 0));
        }
        for (int b = 0; b < S::BUFFERS; ++b) {
            mbar_init(sums_bar(b), 1);
            mbar_init(taken_bar(b), S::EPILOGUE);
        }
        mbar_init(parts_bar, 1);
        abort_word = 0;
        if (g.starve == STARVE_COPY && rank == 0) mbar_expect_more(full_bar(0), 16);
        if (g.starve == STARVE_PARTS) mbar_expect_more(parts_bar, 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"((uint32_t)S::COLUMNS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (g.offsets) list_units<NT, MT>(g, before, at);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    if (blocks > 1) cluster_arrive();          // (waited for in front of the first send: every block runs and has its barriers)

    Units<NT, MT> units(g, before, at);
    bool ok = true;
    int issued = 0;                            // k blocks whose copies (warp 0), or whose MMAs (warp 1), are under way or done
    if (warp == 0) {
        // ---------------- producer: weights by bulk copy, activations by TMA ----------------
        int s = 0;
        uint32_t parity = 1;                                   // (the first lap finds every stage free)
        bool waited = false;
        for (int u = cluster; u < units.total && ok; u += clusters) {
            const Unit unit = units(u);
            const int halves_here = min(MT, g.tiles - unit.tile);
            const uint8_t* w = g.w + ((size_t)((size_t)unit.e * g.tiles + unit.tile) * g.k_blocks + kb_lo) * TILE_BYTES;
            const size_t next_tile = (size_t)g.k_blocks * TILE_BYTES;
            const uint32_t bytes = (uint32_t)halves_here * TILE_BYTES + (uint32_t)unit.width * 128;
            auto weights = [&](int i, int s_) {
                mbar_expect_tx(full_bar(s_), bytes);
                for (int h = 0; h < halves_here; ++h)
                    bulk_copy(base + (uint32_t)s_ * S::STAGE + h * TILE_BYTES, w + h * next_tile + (size_t)i * TILE_BYTES, TILE_BYTES, full_bar(s_));
            };
            // (of one group the first weights are known in front of the wait, and nobody's output)
            int early = 0;
            if (!waited) {
                early = g.offsets ? 0 : min(stages, n_kb);
                if (elect_one())
                    for (int i = 0; i < early; ++i) weights(i, i);
                __syncwarp();
                pdl_wait();
                pdl_trigger();
                waited = true;
            }
            int row[4] = {0, 0, 0, 0};                         // this lane's four of the unit's rows (filled up with its last)
            if (g.order && lane * 4 < unit.width)
#pragma unroll
                for (int q = 0; q < 4; ++q) row[q] = g.order[unit.first + min(lane * 4 + q, unit.here - 1)] / g.top;
            for (int i = 0; i < n_kb; ++i) {
                if (!warp_wait(empty_bar(s), parity, abort_flag, 2 * limit)) { ok = false; break; }
                if (i >= early && elect_one()) weights(i, s);
                __syncwarp();
                const uint32_t dst = base + (uint32_t)s * S::STAGE + MT * TILE_BYTES;
                const int x = (kb_lo + i) * 128;               // (rows are bytes to the tensor map)
                if (g.order) {
                    if (lane * 4 < unit.width) tma_gather4(dst + lane * 512, &map_a, x, row, full_bar(s));
                } else if (elect_one()) {
                    for (int t = 0; t < unit.width; t += 16) tma_load_2d(dst + t * 128, &map_a, x, unit.first + t, full_bar(s));
                }
                __syncwarp();
                ++issued;
                if (++s == stages) { s = 0; parity ^= 1u; }
            }
        }
        if (!waited) {
            pdl_wait();
            pdl_trigger();
        }
        // (the last lap's releases have arrived too before the block may leave: none is on its way to memory that is somebody else's by then)
        for (int j = max(0, issued - stages); ok && j < issued; ++j)
            ok = warp_wait(empty_bar(j % stages), (uint32_t)(j / stages) & 1u, abort_flag, 2 * limit);
        if (!ok && lane == 0) give_up(41);
        if (blocks > 1) cluster_wait();
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        const uint64_t desc_w0 = smem_desc_sw128(base), desc_b0 = smem_desc_sw128(base + MT * TILE_BYTES);
        uint64_t desc_w = desc_w0, desc_b = desc_b0;          // (a stage further is an addition to the address field)
        int s = 0, buffer = 0;
        uint32_t parity = 0, taken = 1;                        // (the first lap finds every buffer free)
        pdl_wait();          // (the copies are complete no sooner, and the time that the kernel in front still takes is not this wait's)
        for (int u = cluster; u < units.total && ok; u += clusters) {
            const Unit unit = units(u);
            const int halves_here = min(MT, g.tiles - unit.tile);
            const uint32_t kind = idesc<FP8>(unit.width);
            for (int i = 0; i < n_kb; ++i) {
                if ((FP8 || i == 0) && !warp_wait(taken_bar(buffer), taken, abort_flag, 2 * limit)) { ok = false; break; }
                if (!warp_wait(full_bar(s), parity, abort_flag, limit)) { ok = false; break; }
                tcgen05_fence_after();
                if (elect_one()) {
                    for (int h = 0; h < halves_here; ++h) {
                        const uint32_t d = tmem_base + (uint32_t)((buffer * MT + h) * NT);
                        const uint64_t dw = desc_w + (uint64_t)(h * (TILE_BYTES >> 4));
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t more = (!FP8 && i > 0) || k > 0;
                            if constexpr (FP8) mma_f8(d, dw + 2 * k, desc_b + 2 * k, kind, more);
                            else tcgen05_mma_bf16(d, dw + 2 * k, desc_b + 2 * k, kind, more);
                        }
                    }
                    tcgen05_commit(empty_bar(s));
                    if (FP8 || i == n_kb - 1) tcgen05_commit(sums_bar(buffer));
                }
                __syncwarp();
                ++issued;
                if (FP8 || i == n_kb - 1)
                    if (++buffer == S::BUFFERS) { buffer = 0; taken ^= 1u; }
                desc_w += S::STAGE >> 4;
                desc_b += S::STAGE >> 4;
                if (++s == stages) { s = 0; parity ^= 1u; desc_w = desc_w0; desc_b = desc_b0; }
            }
        }
        if (!ok && lane == 0) give_up(42);
        if (blocks > 1) cluster_wait();
    } else {
        // ---------------- epilogue: four warps to a tile, TMEM lanes 32 * (warp % 4) = its weight rows ----------------
        const int quad = warp & 3, half = (warp - 2) >> 2, row = quad * 32 + lane, thread = threadIdx.x - 64;
        const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * NT);
        float* park = parks[warp - 2];
        const bool lines = ((uintptr_t)out & 15u) == 0 && (((size_t)g.f.ldo * sizeof(Tout)) & 15u) == 0;
        pdl_wait();          // the token scales, and what is added into, were written by the kernels before
        int buffer = 0, lap = 0;
        uint32_t parity = 0;
        // (in 8 bits a warp whose wait ran out walks on without work: the block's epilogue warps meet at a barrier)
        for (int u = cluster; u < units.total && (FP8 || ok); u += clusters) {
            const Unit unit = units(u);
            const int tile = unit.tile + half, n = tile * 128 + row;
            const bool mine = tile < g.tiles;
            const float bias = g.f.has_bias && n < g.f.N ? g.f.bias[n] : 0.f;
            const bool vec = lines && n - lane + 32 <= g.f.N;
            // what the unit's 16 pairs from 16 c on have come to, from registers (or tensor memory) to out
            auto finish = [&](int c, int lo, int hi) {
                __syncwarp();
                leave<Tout>(g.f, out, park, (size_t)(unit.first + 16 * c), lo, hi, n - lane, vec, lane);
                __syncwarp();
            };
            auto finished = [&](float v) {
                v = g.f.has_bias ? __fadd_rn(v, bias) : v;
                if (g.f.accumulate == EPI_RELU2) {
                    const float z = v < 0.f ? 0.f : v;              // (what is not a number stays so: a maximum would drop it)
                    v = __fmul_rn(z, z);
                }
                return v;
            };
            uint64_t sums[FP8 ? NT / 2 : 1];
            if constexpr (FP8) {
#pragma unroll
                for (int j = 0; j < NT / 2; ++j) sums[j] = 0;
                const int t_row = thread < unit.here ? (g.order ? g.order[unit.first + thread] / g.top : unit.first + thread) : 0;
                const float* sa_row = g.scale_a + (size_t)t_row * g.sa_ld;
                const float* sw_row = g.scale_w + ((size_t)((size_t)unit.e * g.tiles + (mine ? tile : unit.tile)) * 16 + (row >> 3)) * g.sw_ld;
                float4 sa_next = make_float4(0.f, 0.f, 0.f, 0.f), sw_next = *reinterpret_cast<const float4*>(sw_row + (kb_lo & ~3)), sw4 = sw_next;
                if (thread < unit.here) sa_next = *reinterpret_cast<const float4*>(sa_row + (kb_lo & ~3));
                for (int i = 0; i < n_kb; ++i) {
                    const int kb = kb_lo + i;
                    if (i == 0 || (kb & 3) == 0) {
                        // the scales of four k blocks: asked for four blocks ahead, then shared
                        lap ^= 1;
                        sw4 = sw_next;
                        if (thread < NT) {
                            token_scales[lap][0][thread] = sa_next.x;
                            token_scales[lap][1][thread] = sa_next.y;
                            token_scales[lap][2][thread] = sa_next.z;
                            token_scales[lap][3][thread] = sa_next.w;
                        }
                        asm volatile("bar.sync 1, %0;" ::"n"(32 * S::EPILOGUE) : "memory");
                        const int ahead = (kb & ~3) + 4;
                        if (ahead < kb_lo + n_kb) {
                            sw_next = *reinterpret_cast<const float4*>(sw_row + ahead);
                            if (thread < unit.here) sa_next = *reinterpret_cast<const float4*>(sa_row + ahead);
                        }
                    }
                    const int at4 = kb & 3;
                    const float sw = at4 == 0 ? sw4.x : at4 == 1 ? sw4.y : at4 == 2 ? sw4.z : sw4.w;
                    const uint64_t sw2 = pair_of(__float_as_uint(sw), __float_as_uint(sw));
                    const float* sa = token_scales[lap][at4];
                    if (ok) {
                        ok = __all_sync(0xffffffffu, mbar_wait(sums_bar(buffer), parity, abort_flag, 2 * limit));
                        if (!ok && lane == 0) give_up(43);
                    }
                    if (ok) {
                        tcgen05_fence_after();
                        const uint32_t from = taddr + (uint32_t)(buffer * MT * NT);
                        uint32_t v[2][16];
                        tmem_ld(from, v[0]);
                        tmem_ld_wait();
#pragma unroll
                        for (int c = 0; c < CHUNKS; ++c) {
                            if (c > 0 && 16 * c >= unit.width) break;
                            if (c + 1 < CHUNKS && 16 * (c + 1) < unit.width) tmem_ld(from + 16 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const ulonglong2 sa4 = *reinterpret_cast<const ulonglong2*>(sa + 16 * c + 4 * q);
                                uint64_t x = pair_of(v[c & 1][4 * q], v[c & 1][4 * q + 1]), y = pair_of(v[c & 1][4 * q + 2], v[c & 1][4 * q + 3]);
                                asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(sa4.x));
                                asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(y) : "l"(sa4.y));
                                asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sums[8 * c + 2 * q]) : "l"(x), "l"(sw2));
                                asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sums[8 * c + 2 * q + 1]) : "l"(y), "l"(sw2));
                            }
                            if (c + 1 < CHUNKS && 16 * (c + 1) < unit.width) tmem_ld_wait();
                        }
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(taken_bar(buffer));
                    }
                    if (++buffer == S::BUFFERS) { buffer = 0; parity ^= 1u; }
                }
                int mine_lo = 0, mine_end = unit.here;
                if (blocks > 1) {
                    // (one unit a cluster)
                    const int tokens = (unit.here + 7) & ~7, share = g.share;
                    mine_lo = rank * share;
                    const int all_end = min(mine_lo + share, tokens);
                    mine_end = min(all_end, unit.here);
                    if (thread == 0) mbar_expect_tx(parts_bar, (uint32_t)(blocks - 1) * (uint32_t)max(0, all_end - mine_lo) * 512u);
                    cluster_wait();
                    if (ok) {
#pragma unroll
                        for (int q = 0; q < NT / 4; ++q) {
                            const int p = 4 * q / share;
                            if (4 * q < tokens && p != rank) {
                                float v[4];
                                halves(sums[2 * q], v[0], v[1]);
                                halves(sums[2 * q + 1], v[2], v[3]);
                                // of block p's blocks - 1 parts this block's is number `rank`, or rank - 1 if p is below it
                                const uint32_t dst = in_block(base + parts_at + (uint32_t)(rank - (rank > p ? 1 : 0)) * part_bytes + (uint32_t)((4 * q - p * share) / 4) * 2048u + (uint32_t)row * 16, p);
                                asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                                             ::"r"(dst), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
                                               "r"(__float_as_uint(v[3])), "r"(in_block(parts_bar, p))
                                             : "memory");
                            }
                        }
                        if (mine_lo < all_end) ok = __all_sync(0xffffffffu, wait_cluster(parts_bar, 0, abort_flag, 2 * limit));
                    }
                    if (ok) {
                        const uint8_t* parts = aligned + parts_at + (size_t)row * 16;
#pragma unroll
                        for (int q = 0; q < NT / 4; ++q)
                            if (4 * q >= mine_lo && 4 * q < all_end)
                                for (int p = 0; p < blocks - 1; ++p) {
                                    const float4 x = *reinterpret_cast<const float4*>(parts + (size_t)p * part_bytes + (size_t)((4 * q - mine_lo) / 4) * 2048);
                                    float v[4];
                                    halves(sums[2 * q], v[0], v[1]);
                                    halves(sums[2 * q + 1], v[2], v[3]);
                                    sums[2 * q] = pair_of(__float_as_uint(v[0] + x.x), __float_as_uint(v[1] + x.y));
                                    sums[2 * q + 1] = pair_of(__float_as_uint(v[2] + x.z), __float_as_uint(v[3] + x.w));
                                }
                    }
                }
                if (ok && mine)
#pragma unroll 1
                    for (int c = 0; c < CHUNKS; ++c) {
                        const int lo = max(0, mine_lo - 16 * c), hi = min(16, mine_end - 16 * c);
                        if (lo >= hi) continue;
#pragma unroll
                        for (int cc = 0; cc < CHUNKS; ++cc)          // (registers are not indexed: one of these runs)
                            if (cc == c)
#pragma unroll
                                for (int q = 0; q < 8; ++q) {
                                    float a, b;
                                    halves(sums[8 * cc + q], a, b);
                                    park[(2 * q) * 32 + lane] = finished(a);
                                    park[(2 * q + 1) * 32 + lane] = finished(b);
                                }
                        finish(c, lo, hi);
                    }
            } else {
                ok = __all_sync(0xffffffffu, mbar_wait(sums_bar(buffer), parity, abort_flag, 2 * limit));
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t from = taddr + (uint32_t)(buffer * MT * NT);
#pragma unroll 1
                for (int c = 0; 16 * c < unit.here; ++c) {
                    uint32_t v[16];
                    tmem_ld(from + 16 * c, v);
                    tmem_ld_wait();
                    if (16 * (c + 1) >= unit.here) {           // the buffer is the next unit's as soon as its last values are read
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(taken_bar(buffer));
                    }
                    if (mine) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) park[j * 32 + lane] = finished(__uint_as_float(v[j]));
                        finish(c, 0, min(16, unit.here - 16 * c));
                    }
                }
                if (++buffer == S::BUFFERS) { buffer = 0; parity ^= 1u; }
            }
        }
        if (!ok && lane == 0) give_up(43);
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
    if (warp == 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)S::COLUMNS) : "memory");
    }
    // No block of a cluster leaves before everything sent to it is there: its memory is the next block's at once.
    if (blocks > 1) {
        cluster_arrive();
        cluster_wait();
        if (gave_up) drain(parts_bar, 0, now_ns(), limit);
    }
}

// ---- many rows to a group: the rows are the M side -------------------------------------------------------------------------------
// A unit is 128 pairs (the M side) x two tiles of the weight (256 columns). A thread of the epilogue has one pair and the 128 columns of one tile: the
// pair's scale is a register, a tile's scale is one number (of gate and up rows three: a block of 128 up rows may end inside the tile), so a k
// block costs one packed multiply-add for two values and nothing is shared between threads.
constexpr int WIDE_ROWS = 128, WIDE_COLUMNS = 256, WIDE_THREADS = 384, WIDE_PARK = 20;      // (park: rows of 16 values, 20 apart: no two lanes' rows share a bank)
constexpr uint32_t WIDE_STAGE = 3 * TILE_BYTES;
// 384 threads are launched with 168 registers; the copying and issuing warps give of theirs what the sums need
constexpr int WIDE_LAUNCHED = 168, WIDE_FEW = 72, WIDE_MANY = 216;
static_assert(128 * WIDE_FEW + 256 * WIDE_MANY <= WIDE_THREADS * WIDE_LAUNCHED, "what a block was launched with");

// 16 results of a pair (this lane's) -> out, columns from c0 on, through the warp's shared memory, so that a row's results leave together.
template <typename Tout>
__device__ __forceinline__ void leave_rows(const Finish& f, Tout* out, float* park, const float (&v)[16], size_t p0, int rows, int c0, int last, bool vec, int lane) {
    constexpr int PER = 16 / sizeof(Tout), PIECES = 16 / PER;
    __syncwarp();
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<float4*>(park + lane * WIDE_PARK + 4 * q) = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    __syncwarp();
    if (vec && c0 + 16 <= last) {
#pragma unroll
        for (int i = lane; i < 32 * PIECES; i += 32) {
            const int j = i / PIECES, c = i % PIECES * PER;
            if (j >= rows) continue;
            Tout* dst = out + (p0 + j) * f.ldo + c0 + c;
            float x[PER];
#pragma unroll
            for (int q = 0; q < PER; q += 4) *reinterpret_cast<float4*>(x + q) = *reinterpret_cast<const float4*>(park + j * WIDE_PARK + c + q);
            __align__(16) Tout w[PER];
            if (f.accumulate == EPI_ADD) {
                *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(dst);
#pragma unroll
                for (int q = 0; q < PER; ++q) x[q] = __fadd_rn(x[q], to_float(w[q]));
            }
#pragma unroll
            for (int q = 0; q < PER; ++q) w[q] = from_float<Tout>(x[q]);
            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(w);
        }
    } else {
        const int c = lane & 15;
        if (c0 + c < last)
            for (int j = lane >> 4; j < rows; j += 2) {
                Tout* dst = out + (p0 + j) * f.ldo + c0 + c;
                const float x = park[j * WIDE_PARK + c];
                *dst = from_float<Tout>(f.accumulate == EPI_ADD ? __fadd_rn(x, to_float(*dst)) : x);
            }
    }
}

template <bool FP8, bool GLU, typename Tout>
__global__ void __launch_bounds__(WIDE_THREADS, 1)
gemm_grouped_wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ Args g, Tout* __restrict__ out) {
    constexpr int NT = WIDE_ROWS, MT = 2, BUFFERS = 2, COLUMNS = BUFFERS * WIDE_COLUMNS, EPILOGUE = 8;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int before[MAX_GROUPS + 1], at[MAX_GROUPS + 1];
    __shared__ __align__(16) float parks[EPILOGUE][32 * WIDE_PARK];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_word;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int stages = g.stages, n_kb = g.k_blocks;
    const unsigned long long limit = g.limit_us ? g.limit_us * 1000ull : WAIT_NS;
    const uint32_t bars = base + (uint32_t)stages * WIDE_STAGE;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (stages + s); };
    auto sums_bar = [&](int b) { return bars + 16u * stages + 8u * b; };
    auto taken_bar = [&](int b) { return bars + 16u * stages + 8u * (BUFFERS + b); };
    volatile int* abort_flag = &abort_word;
    auto give_up = [&](int code) {
        atomicCAS(g.error_word, 0, code);
        __threadfence();               // (before anybody follows the flag and has a code of his own)
        *abort_flag = 1;
    };
    const int warp = uniform_warp(), lane = threadIdx.x & 31, blocks = (int)gridDim.x;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1 + (g.starve == STARVE_RELEASE && s == 0));
        }
        for (int b = 0; b < BUFFERS; ++b) {
            mbar_init(sums_bar(b), 1);
            mbar_init(taken_bar(b), EPILOGUE);
        }
        abort_word = 0;
        if (g.starve == STARVE_COPY && blockIdx.x == 0) mbar_expect_more(full_bar(0), 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"((uint32_t)COLUMNS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (g.offsets) list_units<NT, MT>(g, before, at);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = tmem_base_slot;

    Units<NT, MT> units(g, before, at);
    bool ok = true;
    int issued = 0;                            // k blocks whose copies (warp 0), or whose MMAs (warp 1), are under way or done
    if (warp < 4) {
        if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(WIDE_FEW));
        if (warp == 0) {
            // ---------------- producer ----------------
            int s = 0;
            uint32_t parity = 1;                                   // (the first lap finds every stage free)
            bool waited = false;
            for (int u = (int)blockIdx.x; u < units.total && ok; u += blocks) {
                const Unit unit = units(u);
                const int halves_here = min(MT, g.tiles - unit.tile);
                const uint8_t* w = g.w + (size_t)((size_t)unit.e * g.tiles + unit.tile) * n_kb * TILE_BYTES;
                const size_t next_tile = (size_t)n_kb * TILE_BYTES;
                const uint32_t bytes = (uint32_t)halves_here * TILE_BYTES + (uint32_t)unit.width * 128;
                auto weights = [&](int i, int s_) {
                    mbar_expect_tx(full_bar(s_), bytes);
                    for (int h = 0; h < halves_here; ++h)
                        bulk_copy(base + (uint32_t)s_ * WIDE_STAGE + h * TILE_BYTES, w + h * next_tile + (size_t)i * TILE_BYTES, TILE_BYTES, full_bar(s_));
                };
                // (of one group the first weights are known in front of the wait, and nobody's output)
                int early = 0;
                if (!waited) {
                    early = g.offsets ? 0 : min(stages, n_kb);
                    if (elect_one())
                        for (int i = 0; i < early; ++i) weights(i, i);
                    __syncwarp();
                    pdl_wait();
                    pdl_trigger();
                    waited = true;
                }
                int row[4] = {0, 0, 0, 0};                         // this lane's four of the unit's rows (filled up with its last)
                if (g.order && lane * 4 < unit.width)
#pragma unroll
                    for (int q = 0; q < 4; ++q) row[q] = g.order[unit.first + min(lane * 4 + q, unit.here - 1)] / g.top;
                for (int i = 0; i < n_kb; ++i) {
                    if (!warp_wait(empty_bar(s), parity, abort_flag, 2 * limit)) { ok = false; break; }
                    if (i >= early && elect_one()) weights(i, s);
                    __syncwarp();
                    const uint32_t dst = base + (uint32_t)s * WIDE_STAGE + MT * TILE_BYTES;
                    const int x = i * 128;               // (rows are bytes to the tensor map)
                    if (g.order) {
                        if (lane * 4 < unit.width) tma_gather4(dst + lane * 512, &map_a, x, row, full_bar(s));
                    } else if (elect_one()) {
                        for (int t = 0; t < unit.width; t += 16) tma_load_2d(dst + t * 128, &map_a, x, unit.first + t, full_bar(s));
                    }
                    __syncwarp();
                    ++issued;
                    if (++s == stages) { s = 0; parity ^= 1u; }
                }
            }
            if (!waited) {
                pdl_wait();
                pdl_trigger();
            }
            // (the last lap's releases have arrived too before the block may leave: none is on its way to memory that is somebody else's by then)
            for (int j = max(0, issued - stages); ok && j < issued; ++j)
                ok = warp_wait(empty_bar(j % stages), (uint32_t)(j / stages) & 1u, abort_flag, 2 * limit);
            if (!ok && lane == 0) give_up(41);
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            const uint64_t desc_w0 = smem_desc_sw128(base), desc_a0 = smem_desc_sw128(base + MT * TILE_BYTES);
            uint64_t desc_w = desc_w0, desc_a = desc_a0;          // (a stage further is an addition to the address field)
            int s = 0, buffer = 0;
            uint32_t parity = 0, taken = 1;                        // (the first lap finds every buffer free)
            pdl_wait();          // (the copies are complete no sooner, and the time that the kernel in front still takes is not this wait's)
            for (int u = (int)blockIdx.x; u < units.total && ok; u += blocks) {
                const Unit unit = units(u);
                const uint32_t kind = idesc<FP8>(128 * min(MT, g.tiles - unit.tile));
                for (int i = 0; i < n_kb; ++i) {
                    if ((FP8 || i == 0) && !warp_wait(taken_bar(buffer), taken, abort_flag, 2 * limit)) { ok = false; break; }
                    if (!warp_wait(full_bar(s), parity, abort_flag, limit)) { ok = false; break; }
                    tcgen05_fence_after();
                    if (elect_one()) {
                        const uint32_t d = tmem_base + (uint32_t)(buffer * WIDE_COLUMNS);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t more = (!FP8 && i > 0) || k > 0;
                            if constexpr (FP8) mma_f8(d, desc_a + 2 * k, desc_w + 2 * k, kind, more);
                            else tcgen05_mma_bf16(d, desc_a + 2 * k, desc_w + 2 * k, kind, more);
                        }
                        tcgen05_commit(empty_bar(s));
                        if (FP8 || i == n_kb - 1) tcgen05_commit(sums_bar(buffer));
                    }
                    __syncwarp();
                    ++issued;
                    if (FP8 || i == n_kb - 1)
                        if (++buffer == BUFFERS) { buffer = 0; taken ^= 1u; }
                    desc_w += WIDE_STAGE >> 4;
                    desc_a += WIDE_STAGE >> 4;
                    if (++s == stages) { s = 0; parity ^= 1u; desc_w = desc_w0; desc_a = desc_a0; }
                }
            }
            if (!ok && lane == 0) give_up(42);
        }
    } else {
        // ---------------- epilogue: TMEM lanes 32 * (warp % 4) = the unit's pairs, warps 4..7 its first tile, 8..11 its second ----------------
        if constexpr (FP8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(WIDE_MANY));
        const int quad = warp & 3, half = (warp - 4) >> 2, token = quad * 32 + lane;
        const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * 128);
        float* park = parks[warp - 4];
        const bool vec = ((uintptr_t)out & 15u) == 0 && (((size_t)g.f.ldo * sizeof(Tout)) & 15u) == 0;
        const int last = GLU ? g.f.N >> 1 : g.f.N;
        pdl_wait();          // the token scales, and what is added into, were written by the kernels before
        int buffer = 0;
        uint32_t parity = 0;
        for (int u = (int)blockIdx.x; u < units.total && ok; u += blocks) {
            const Unit unit = units(u);
            const int tile = unit.tile + half, rows = min(32, unit.here - quad * 32), c_tile = tile * (GLU ? 64 : 128);
            const bool mine = tile < g.tiles && rows > 0;
            const size_t p0 = (size_t)(unit.first + quad * 32);
            // 32 columns of this lane's pair (a quarter of the tile) to results
            auto finish = [&](float (&v)[32], int c) {
                if constexpr (GLU) {
                    float units16[16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float eight[8];
                        glu_units<8, true>(g.f.glu, [&](int q) { return v[16 * h + q]; }, [&](int q) { return v[16 * h + 8 + q]; }, 1.f, eight);
#pragma unroll
                        for (int q = 0; q < 8; ++q) units16[8 * h + q] = eight[q];
                    }
                    if (c_tile + 16 * c < last) leave_rows<Tout>(g.f, out, park, units16, p0, rows, c_tile + 16 * c, last, vec, lane);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int c0 = c_tile + 32 * c + 16 * h;
                        if (c0 >= last) break;
                        float x[16];
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            x[q] = v[16 * h + q];
                            if (g.f.has_bias && c0 + q < last) x[q] = __fadd_rn(x[q], g.f.bias[c0 + q]);
                            if (g.f.accumulate == EPI_RELU2) {
                                const float z = x[q] < 0.f ? 0.f : x[q];              // (what is not a number stays so: a maximum would drop it)
                                x[q] = __fmul_rn(z, z);
                            }
                        }
                        leave_rows<Tout>(g.f, out, park, x, p0, rows, c0, last, vec, lane);
                    }
                }
            };
            if constexpr (FP8) {
                uint64_t sums[64];
#pragma unroll
                for (int j = 0; j < 64; ++j) sums[j] = 0;
                const int t_row = token < unit.here ? (g.order ? g.order[unit.first + token] / g.top : unit.first + token) : -1;
                const float* sa_row = g.scale_a + (size_t)max(t_row, 0) * g.sa_ld;
                const float* sw_row = g.scale_w + (size_t)((size_t)unit.e * g.tiles + (tile < g.tiles ? tile : unit.tile)) * 16 * g.sw_ld;
                // of gate and up rows in eights: the gates' scale, and the up rows' in front of and behind the edge of their block
                const int edge = GLU ? (128 - ((last + c_tile) & 127)) >> 3 : 0;
                float4 sa4 = make_float4(0.f, 0.f, 0.f, 0.f), sa_next = sa4, sw4[GLU ? 3 : 1], sw_next[GLU ? 3 : 1];
                auto ask = [&](int kb) {
                    if (t_row >= 0) sa_next = *reinterpret_cast<const float4*>(sa_row + kb);
                    sw_next[0] = *reinterpret_cast<const float4*>(sw_row + kb);
                    if constexpr (GLU) {
                        sw_next[1] = *reinterpret_cast<const float4*>(sw_row + g.sw_ld + kb);
                        sw_next[2] = *reinterpret_cast<const float4*>(sw_row + 15 * g.sw_ld + kb);
                    }
                };
                ask(0);
                for (int kb = 0; kb < n_kb; ++kb) {
                    if ((kb & 3) == 0) {
                        sa4 = sa_next;
#pragma unroll
                        for (int q = 0; q < (GLU ? 3 : 1); ++q) sw4[q] = sw_next[q];
                        if (kb + 4 < n_kb) ask(kb + 4);
                    }
                    const int at4 = kb & 3;
                    auto of4 = [&](const float4& f4) { return at4 == 0 ? f4.x : at4 == 1 ? f4.y : at4 == 2 ? f4.z : f4.w; };
                    const float sa = of4(sa4);
                    uint64_t scale[GLU ? 3 : 1];
#pragma unroll
                    for (int q = 0; q < (GLU ? 3 : 1); ++q) {
                        const uint32_t both = __float_as_uint(__fmul_rn(sa, of4(sw4[q])));
                        scale[q] = pair_of(both, both);
                    }
                    ok = __all_sync(0xffffffffu, mbar_wait(sums_bar(buffer), parity, abort_flag, 2 * limit));
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t from = taddr + (uint32_t)(buffer * WIDE_COLUMNS);
                    uint32_t v[2][16];
                    tmem_ld(from, v[0]);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        if (c < 7) tmem_ld(from + 16 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const uint64_t x = pair_of(v[c & 1][2 * q], v[c & 1][2 * q + 1]);
                            const uint64_t by = !GLU || q < 4 ? scale[0] : c < edge ? scale[GLU ? 1 : 0] : scale[GLU ? 2 : 0];
                            asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sums[8 * c + q]) : "l"(x), "l"(by));
                        }
                        if (c < 7) tmem_ld_wait();
                    }
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(taken_bar(buffer));
                    if (++buffer == BUFFERS) { buffer = 0; parity ^= 1u; }
                }
                if (ok && mine)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float v[32];
#pragma unroll
                        for (int q = 0; q < 16; ++q) halves(sums[16 * c + q], v[2 * q], v[2 * q + 1]);
                        finish(v, c);
                    }
            } else {
                ok = __all_sync(0xffffffffu, mbar_wait(sums_bar(buffer), parity, abort_flag, 2 * limit));
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t from = taddr + (uint32_t)(buffer * WIDE_COLUMNS);
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[32];
                    tmem_ld_32x32b_x32(from + 32 * c, r);
                    tmem_ld_wait();
                    if (c == 3) {           // the buffer is the next unit's as soon as its last values are read
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(taken_bar(buffer));
                    }
                    float v[32];
#pragma unroll
                    for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(r[q]);
                    if (mine) finish(v, c);
                }
                if (++buffer == BUFFERS) { buffer = 0; parity ^= 1u; }
            }
        }
        if (!ok && lane == 0) give_up(43);
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
    if (warp == 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)COLUMNS) : "memory");
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------

// Rows of `bytes` bytes, `ld` bytes apart, read in boxes of box_rows x 128 bytes with the 128-byte swizzle (box_rows 1: gathers of four).
int rows_map_for(const void* ptr, long long rows, long long bytes, long long ld, int box_rows, CUtensorMap* out) {
    static std::unordered_map<MapKey, CUtensorMap, MapKeyHash> cache;
    static std::mutex mu;
    const MapKey key{ptr, rows, bytes, ld, box_rows};
    std::lock_guard<std::mutex> lock(mu);
    auto it = cache.find(key);
    if (it != cache.end()) {
        *out = it->second;
        return JLLM_OK;
    }
    EncodeTiledFn fn = encode_fn();
    if (!fn) return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: the driver does not offer cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    CUtensorMap map;
    const CUresult r = fn(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: cuTensorMapEncodeTiled failed (%d) for [%lld, %lld] bytes, ld %lld", (int)r, rows, bytes, ld);
    if (cache.size() > 4096) cache.clear();
    cache.emplace(key, map);
    *out = map;
    return JLLM_OK;
}

// How a product is cut: pairs of a span, tiles of a unit, blocks of a cluster, blocks that an SM is to hold.
struct Cut {
    int nt, mt, blocks, per_sm;
};
// (what stands for a cut in one number, for tests)
Cut cut_of(int code) { return {code / 1000, code / 100 % 10, code % 10, code / 10 % 10}; }

struct Product {
    Args args;
    const CUtensorMap* map;
    int pairs, out_dtype;
    void* out;
    cudaStream_t stream;
};

// What a kernel is to the launcher: pairs and tiles of a unit, a stage's bytes, buffers and columns of tensor memory, threads.
struct Kind {
    int nt, mt;
    uint32_t stage;
    int buffers, columns, threads;
    bool clusters;
};

template <typename Tout>
int launch(void (*kern)(const CUtensorMap, const Args, Tout*), const Kind& kind, size_t own, const Product& p, const Cut& cut) {
    Args g = p.args;
    const int sms = jllm_device_sm_count(), tiles = (g.tiles + kind.mt - 1) / kind.mt;
    if (sms <= 0 || own == 0) return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: the device does not say how many SMs it has, or what the kernel holds");
    // (of groups: every group that has pairs ends one span that is not full)
    const long long spans = g.offsets ? (long long)p.pairs / kind.nt + (g.groups < p.pairs ? g.groups : p.pairs) : ((long long)g.rows + kind.nt - 1) / kind.nt;
    const long long units = spans * tiles;
    JLLM_REQUIRE(units * cut.blocks < BLOCK_MOST, "gemm_grouped: %lld units of work", units);
    g.blocks = cut.blocks;
    g.share = cut.blocks > 1 ? ((g.rows + 7) / 8 + cut.blocks - 1) / cut.blocks * 8 : 0;
    JLLM_REQUIRE(cut.blocks >= 1 && cut.blocks <= 8 && cut.blocks <= g.k_blocks && (cut.blocks == 1 || (kind.clusters && !g.offsets && g.rows <= kind.nt)),
                 "gemm_grouped: no clusters of %d blocks for such a product", cut.blocks);
    // An SM has 228 KB, a block 227 at most; each block's last KB is the system's, `own` what the kernel holds by itself.
    const size_t parts = (size_t)(cut.blocks - 1) * g.share * 512, fixed = 1024 + 8 * (2 * kind.buffers + 1) + 64, each = kind.stage + 16;
    const size_t all = cut.per_sm == 1 ? 227 * 1024 : 113 * 1024;
    JLLM_REQUIRE((cut.per_sm == 1 || cut.per_sm == 2) && kind.columns * cut.per_sm <= 512 && own + fixed + parts + 2 * each <= all,
                 "gemm_grouped: %d blocks of such a product on an SM", cut.per_sm);
    int stages = (int)((all - own - fixed - parts) / each);
    if (!g.offsets && cut.blocks == 1) {
        // (no more than a block has k blocks)
        const long long most = (units + (long long)sms * cut.per_sm - 1) / ((long long)sms * cut.per_sm) * g.k_blocks;
        if (stages > most) stages = most < 2 ? 2 : (int)most;
    }
    g.stages = stages;
    // Blocks that wait for one another must not wait for tensor memory that others hold who wait in turn: a cluster's block takes all of an SM's
    // shared memory, so none that holds columns is beside it.
    const size_t smem = stages * each + parts + fixed;
    if (jllm_allow_smem((const void*)kern, smem) != cudaSuccess)
        return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: %zu bytes of shared memory refused", smem);
    const long long at_once = (long long)sms * cut.per_sm, grid = cut.blocks > 1 ? units * cut.blocks : units < at_once ? units : at_once;
    JLLM_REQUIRE(g.starve == STARVE_NOTHING || (grid <= 64 && (g.starve != STARVE_PARTS || cut.blocks > 1)),
                 "gemm_grouped: the starved product of the wait test has at most 64 blocks, and a cluster where parts are missed");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kind.threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = p.stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cut.blocks > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cut.blocks;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    if (jllm_launch_overlaps(smem, LAUNCH_DEPENDENT)) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaLaunchKernelEx(&cfg, kern, *p.map, g, static_cast<Tout*>(p.out));
    return jllm_check_launch("gemm_grouped");
}

// What a kernel holds of shared memory by itself; 0 if the driver does not say, or if its threads are launched with fewer registers than `least`.
size_t own_smem(const void* kern, int least = 0) {
    cudaFuncAttributes a{};
    if (cudaFuncGetAttributes(&a, kern) == cudaSuccess) return a.numRegs >= least ? a.sharedSizeBytes : 0;
    cudaGetLastError();
    return 0;
}

template <bool FP8, int NT, typename Tout>
int launch_narrow(const Product& p, const Cut& cut) {
    using S = Shape<FP8, NT, 1>;
    auto kern = gemm_grouped_kernel<FP8, NT, 1, Tout>;
    static const size_t own = own_smem((const void*)kern);
    return launch<Tout>(kern, Kind{NT, 1, S::STAGE, S::BUFFERS, S::COLUMNS, S::THREADS, FP8}, own, p, cut);
}
template <bool FP8, bool GLU, typename Tout>
int launch_wide(const Product& p, const Cut& cut) {
    auto kern = gemm_grouped_wide_kernel<FP8, GLU, Tout>;
    static const size_t own = own_smem((const void*)kern, FP8 ? WIDE_LAUNCHED : 0);          // (what the warps hand over has to be there)
    return launch<Tout>(kern, Kind{WIDE_ROWS, 2, WIDE_STAGE, 2, 512, WIDE_THREADS, false}, own, p, cut);
}

template <bool FP8, typename Tout>
int launch_cut(const Product& p, const Cut& cut) {
    if (cut.nt == 16 && cut.mt == 1) return launch_narrow<FP8, 16, Tout>(p, cut);
    if (cut.nt == 32 && cut.mt == 1) return launch_narrow<FP8, 32, Tout>(p, cut);
    if (cut.nt == 64 && cut.mt == 1) return launch_narrow<FP8, 64, Tout>(p, cut);
    if (cut.nt == WIDE_ROWS && cut.mt == 2) return p.args.f.glu ? launch_wide<FP8, true, Tout>(p, cut) : launch_wide<FP8, false, Tout>(p, cut);
    return jllm_fail(JLLM_BAD_ARGUMENT, "gemm_grouped: no kernel for spans of %d pairs and %d tiles", cut.nt, cut.mt);
}

Cut choose(bool fp8, int groups, int pairs, int tiles, int k_blocks) {
    const int sms = jllm_device_sm_count(), asked = groups < pairs ? groups : pairs, mean = (pairs + asked - 1) / asked;
    Cut cut{128, 1, 1, 1};
    if (groups == 1) {
        cut.nt = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : 128;
        const int units = tiles * ((mean + cut.nt - 1) / cut.nt);
        if (fp8 && cut.nt <= 64 && units < sms) {
            cut.blocks = sms / units;
            if (cut.blocks > 8) cut.blocks = 8;
            while (cut.blocks > 1 && k_blocks / cut.blocks < 2) --cut.blocks;
        }
        if (cut.nt == 128) cut.mt = 2;
    } else {
        cut.nt = mean <= 6 ? 16 : mean <= 20 ? 32 : mean <= 48 ? 64 : 128;
        if (cut.nt == 128) cut.mt = 2;
    }
    return cut;
}

// A test of the waits: what the next product of this thread is to miss, and how long its waits last.
struct Starve {
    int what, limit_us;
};
thread_local Starve g_starve_next = {STARVE_NOTHING, 0};

}  // namespace

int* jllm_gemm_error_word();

// A test of the bounded waits: the NEXT product of this thread has waits of `limit_us` microseconds, and with `what` 1 a copy's barrier that
// expects more than comes, with 2 a stage that is never released, with 3 a part that no block of the cluster sends (0: the limit alone). It
// returns, raises the error word and leaves the device usable.
JLLM_EXPORT int jllm_gemm_grouped_starve_next(int what, int limit_us) {
    JLLM_REQUIRE(what >= STARVE_NOTHING && what <= STARVE_PARTS && limit_us >= 1 && limit_us <= 1000000, "gemm_grouped_starve_next: %d, %d us", what, limit_us);
    g_starve_next = {what, limit_us};
    return JLLM_OK;
}

// `rows`: what is multiplied (of e4m3, with the scales), [M, K]; `weight`: the packed weight(s) [N, K]; `groups`: null (one weight, out [M, N]) or
// the groups of pairs (out [pairs, N], of which the rows behind the last pair stay as they were), `by_pair` whether `rows` are the pairs'
// already. With `swiglu_word` out has N / 2 columns. `cut` (tests): see Cut; 0 as the sizes have it.
JLLM_EXPORT int jllm_gemm_grouped(const BlockRows* rows, const BlockWeight* weight, const RowGroupsView* groups, int by_pair, const void* bias,
                                  int bias_dtype, void* out, int out_dtype, int ldo, int accumulate, int swiglu_word, int cut_code, cudaStream_t stream) {
    const Starve starve = g_starve_next;
    g_starve_next = {STARVE_NOTHING, 0};
    const bool fp8 = weight->scale != nullptr;
    const int M = rows->rows, K = rows->cols, N = weight->rows, bytes = fp8 ? 1 : 2, per_block = 128 / bytes;
    const long long pairs = groups ? (long long)groups->rows * groups->top : M;
    JLLM_REQUIRE(M == 0 || (rows->scale != nullptr) == fp8, "gemm_grouped: rows and weight are both e4m3 with scales or both bfloat16");
    JLLM_REQUIRE(M >= 0 && M <= BLOCK_MOST && N >= 1 && N <= BLOCK_MOST && K >= 1 && K == weight->cols && pairs <= BLOCK_MOST,
                 "gemm_grouped: M=%d N=%d K=%d against a weight of %d, %lld pairs", M, N, K, weight->cols, pairs);
    JLLM_REQUIRE(weight->k_blocks == (K + per_block - 1) / per_block, "gemm_grouped: the packed weight has %d k blocks, K=%d needs %d", weight->k_blocks,
                 K, (K + per_block - 1) / per_block);
    JLLM_REQUIRE(rows->stride >= (long long)K * bytes && rows->stride % 16 == 0 && ((uintptr_t)rows->data % 16) == 0 && ((uintptr_t)weight->data % 16) == 0,
                 "gemm_grouped: rows and weights begin at multiples of 16 bytes (%lld bytes a row, K=%d)", rows->stride, K);
    JLLM_REQUIRE(!fp8 || (rows->scale_ld % 4 == 0 && rows->scale_ld >= weight->k_blocks && weight->scale_ld % 4 == 0 && weight->scale_ld >= weight->k_blocks &&
                          ((uintptr_t)rows->scale % 16) == 0 && ((uintptr_t)weight->scale % 16) == 0),
                 "gemm_grouped: scales lie in rows of whole fours (%d and %d for %d blocks)", rows->scale_ld, weight->scale_ld, weight->k_blocks);
    JLLM_REQUIRE(groups ? groups->groups == weight->groups && groups->groups >= 1 && groups->groups <= MAX_GROUPS && (by_pair ? pairs : groups->rows) == M
                        : weight->groups == 1,
                 "gemm_grouped: %d weights (1 to %d), %d rows and the groups of another product", weight->groups, MAX_GROUPS, M);
    JLLM_REQUIRE(accumulate >= EPI_STORE && accumulate <= EPI_RELU2 && (!groups || (!accumulate && !bias)), "gemm_grouped: accumulate=%d, groups take neither it nor a bias", accumulate);
    JLLM_REQUIRE((swiglu_word != 0) == (weight->glu != 0) && (!swiglu_word || (N % 16 == 0 && !bias && !accumulate)),
                 "gemm_grouped: a gated unit needs a weight packed for it, no bias and no accumulation (N=%d)", N);
    JLLM_REQUIRE(ldo >= (swiglu_word ? N / 2 : N), "gemm_grouped: ldo=%d < N=%d", ldo, N);
    if (pairs == 0) return JLLM_OK;
    int* error_word = jllm_gemm_error_word();
    if (!error_word) return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: no error word");
    const bool gather = groups && !by_pair;
    CUtensorMap map;
    const int rc = rows_map_for(rows->data, M, (long long)K * bytes, rows->stride, gather ? 1 : 16, &map);
    if (rc != JLLM_OK) return rc;
    Product p;
    p.args = Args{static_cast<const uint8_t*>(weight->data), weight->scale, rows->scale, groups ? groups->offsets : nullptr, gather ? groups->order : nullptr,
                  weight->scale_ld, rows->scale_ld, weight->groups, groups ? groups->top : 1, M, (N + 127) / 128, weight->k_blocks,
                  Finish{VecRef{bias, bias_dtype}, (int)(bias != nullptr), ldo, accumulate, N, swiglu_word}, 0, 1, 0, starve.what, starve.limit_us, error_word};
    p.map = &map, p.pairs = (int)pairs, p.out_dtype = out_dtype, p.out = out, p.stream = stream;
    const Cut cut = cut_code ? cut_of(cut_code) : choose(fp8, groups ? weight->groups : 1, (int)pairs, p.args.tiles, weight->k_blocks);
    if (fp8) return out_dtype == JLLM_F32 ? launch_cut<true, float>(p, cut) : launch_cut<true, __nv_bfloat16>(p, cut);
    return out_dtype == JLLM_F32 ? launch_cut<false, float>(p, cut) : launch_cut<false, __nv_bfloat16>(p, cut);
}
