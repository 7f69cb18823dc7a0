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
// 16 KB.
//
// The blocks stay: block b takes the units b, b + blocks, ... of a list that every block reckons by itself from the offsets (the host does not
// know them). One warp brings weights (bulk copies) and rows into a ring that runs on over the units, one issues the MMAs, the others take the sums
// from tensor memory. So the copies of the next unit are under way while this one ends. Rows that lie together come by TMA boxes; rows that are
// fetched from all over by 16-byte asynchronous copies of whole warps, four rows an instruction (gathers of four rows by TMA took 30 ns each and
// an SM: 16,384 pairs of 128 groups against 1,536 x 2,048, bfloat16, 281 us; now 175, and 151 of rows that lie together).
//
// In 8 bits the sums of ONE k block are made by the tensor cores (float32) and lie in one of several buffers in tensor memory; the epilogue warps
// multiply them by both scales and add them into float32 registers. The scales of a block are float32 numbers of any value: the hardware's own
// block scales are powers of two for 32 values each.
//
// Two kernels. NARROW, groups of few rows: the weight rows are the M side of the MMAs and up to 64 rows of a group, filled up to a multiple of 16, the
// N side, so that of many small groups nothing is wasted on a side of 128. WIDE, groups of many: 128 rows are the M side and two tiles of the weight the
// N side. Which one, and how it is cut, follows from counts that are fitted to measured sizes (`choose`).
//
// What bounds them. Few rows: memory. Eight rows of eight choices among 128 weights of 1,536 x 2,048 (bfloat16, 49 asked) 48 us for 308 MB (6.4 TB/s, 0.98 of the
// measured copy), sixteen rows in 8 bits 46 us for 250 MB; one row in 8 bits against 24,576 x 4,096 18 us (5.6 TB/s), against 4,096 x 4,096 6.4 us (launch, scales, ring,
// the cluster's parts: about 4 us beside the stream). Many rows: bfloat16 groups are near memory too (2,048 rows, 128 groups of 1,536 x 2,048: 175 us for 128 of
// bytes). In 8 bits it is the way of a k block from the tensor cores to the epilogue's registers and back, over two buffers, which are all of tensor
// memory: some 1,000 cycles a k block and SM where its MMAs (128 x 256 x 128) take 512. By cycle counts a warp of the sums spends 390 on its loads of tensor memory and
// multiply-adds (256 are the float32 units' least), 140 on waiting, the rest on scales, barriers and, spread over a unit's k blocks, its results; the issuing warp waits 450 to 600
// for a buffer and 90 for copies. 2,048 x 24,576 x 4,096 take 213 to 227 us (1.8 to 1.9 PFLOP/s), 264 one behind the other for long (the power limit). Measured slower: the two tiles of a k block
// handed over apart (1 to 2%), eight warps of twice the columns, k blocks unrolled by four. Also slower: the last round's units shared out by weight rows (8-bit down of
// 2,048 rows 118 us for 102).
//
// The waits on barriers in shared memory end by the clock and raise the products' error word (41: the producer, 42: the MMAs, 43: the epilogue).
#include "fp8_view.h"
#include "tcgen05_common.cuh"

#include <atomic>
#include <cmath>

namespace {

using namespace tc;

constexpr int TILE_BYTES = 128 * 128;
constexpr int MAX_GROUPS = 1024;

struct Finish {
    VecRef bias;
    int has_bias, ldo, accumulate, N, glu;
};

struct Args {
    const uint8_t *w, *a;
    const float *scale_w, *scale_a;       // [groups, tiles * 16, sw_ld] and [rows, sa_ld]: multiples of four values a row
    const int *offsets, *order;           // null: one group of `rows`; null: a pair's row is the pair
    int sw_ld, sa_ld;
    int groups, top, rows, pairs, tiles, k_blocks;
    int spans, span;                      // of one group: spans of so many rows
    int row_bytes, row_step;              // of `a`: bytes that count, and 16-byte pieces from row to row
    Finish f;
    int stages, blocks, share;            // blocks of a cluster, tokens that each of them finishes
    int box;                              // rows that one copy brings, of rows that lie together
    int starve, limit_us;                 // a test of the waits (below); 0, 0
    int* error_word;
};
enum : int { STARVE_NOTHING = 0, STARVE_COPY = 1, STARVE_RELEASE = 2, STARVE_PARTS = 3 };

// A unit: group e's weight from `tile` on against `here` pairs from `first` on, filled up to `width`.
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

// ---- what a kernel is made of: rows and tiles of a unit, buffers of sums in tensor memory (in 8 bits one k block's, else a unit's), warps ----
template <bool FP8, int NT>
struct Narrow {
    // (in 8 bits a buffer has two k blocks' sums: what barriers and waits cost is paid for two;
    // and there are as many as half of tensor memory holds, so that the ring does not wait while the first scales come)
    static constexpr int ROWS = NT, TILES = 1, TOGETHER = FP8 ? 2 : 1, COLUMNS = TOGETHER * NT, BUFFERS = FP8 ? 256 / COLUMNS : 2,
                         TMEM = BUFFERS * COLUMNS < 32 ? 32 : BUFFERS * COLUMNS;
    // four warps have the tile's weight rows; with 32 rows and more two sets of them share the rows
    static constexpr int SETS = NT >= 32 ? 2 : 1, EPILOGUE = 4 * SETS, FIRST = 2, THREADS = 32 * (FIRST + EPILOGUE);
    static constexpr bool ONE = FP8;                           // products of one weight without groups: in 8 bits alone
    static constexpr bool CLUSTERS = FP8 && NT <= 32;          // (the parts of 64 rows leave no room for a ring beside another block)
    static constexpr int GATHER = 0, GATHER_WARPS = 1, GATHER_ROWS = NT;          // the producer fetches rows itself
    static constexpr uint32_t STAGE = TILES * TILE_BYTES + NT * 128;
};
template <bool FP8>
struct Wide {
    static constexpr int ROWS = 128, TILES = 2, TOGETHER = 1, COLUMNS = 256, BUFFERS = 2, TMEM = BUFFERS * COLUMNS;
    // four warps have the rows; four sets of them share the 256 columns
    static constexpr int SETS = 4, EPILOGUE = 4 * SETS, FIRST = 4, THREADS = 32 * (FIRST + EPILOGUE);
    static constexpr bool ONE = FP8;
    static constexpr int GATHER = 2, GATHER_WARPS = 2, GATHER_ROWS = 64;
    static constexpr uint32_t STAGE = TILES * TILE_BYTES + ROWS * 128;
    // The threads are launched with 96 registers; the copying and issuing warps give of theirs what the sums need.
    static constexpr int LAUNCHED = 96, FEW = 64, MANY = 104;
    static_assert(32 * (FIRST * FEW + EPILOGUE * MANY) <= THREADS * LAUNCHED, "what a block was launched with");
};
constexpr int FETCHED = 2;          // stages of fetched rows that a warp has under way behind the newest

// A block's ring and barriers in shared memory.
template <class S>
struct Ring {
    uint32_t base, bars;
    int stages;
    __device__ __forceinline__ uint32_t stage(int s) const { return base + (uint32_t)s * S::STAGE; }
    __device__ __forceinline__ uint32_t rows(int s) const { return stage(s) + S::TILES * TILE_BYTES; }
    __device__ __forceinline__ uint32_t full(int s) const { return bars + 8u * s; }
    __device__ __forceinline__ uint32_t empty(int s) const { return bars + 8u * (stages + s); }
    __device__ __forceinline__ uint32_t sums(int b) const { return bars + 16u * stages + 8u * b; }                      // a buffer's sums are there
    __device__ __forceinline__ uint32_t taken(int b) const { return bars + 16u * stages + 8u * (S::BUFFERS + b); }     // ... have been read
    __device__ __forceinline__ uint32_t parts() const { return bars + 16u * stages + 16u * S::BUFFERS; }
};
// ... behind them the two lists of groups (Units)
template <class S>
constexpr size_t fixed_smem() { return 1024 + 8 * (2 * S::BUFFERS + 1) + 64; }

// Units in front of every group, by the whole block (a lane has 32 neighbouring groups at most); a __syncthreads has to follow. Offsets are a kernel's output, which
// the host cannot check: a larger step's that were not filled anew are cut off at the pairs there are, and numbers that do not ascend from 0 on are no pairs, so
// that whatever they are nothing outside the rows and the result is touched.
template <class S>
__device__ __forceinline__ void list_units(const Args& g, int* before, int* at) {
    pdl_wait();          // (the offsets are the kernel in front's)
    for (int i = threadIdx.x; i <= g.groups; i += blockDim.x) at[i] = min(g.offsets[i], g.pairs);
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const int lane = threadIdx.x, each = (g.groups + 31) / 32, lo = min(lane * each, g.groups), hi = min(lo + each, g.groups);
    int tiles = (g.tiles + S::TILES - 1) / S::TILES, sum = 0;
    bool wrong = false;
    for (int i = lo; i < hi; ++i) {
        const int here = at[i], next = at[i + 1];
        wrong |= here < 0 || next < here;
        sum += wrong ? 0 : (next - here + S::ROWS - 1) / S::ROWS * tiles;
    }
    if (__any_sync(0xffffffffu, wrong)) sum = tiles = 0;
    int run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int left = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += left;
    }
    run -= sum;
    for (int i = lo; i < hi; ++i) {
        before[i] = run;
        run += (at[i + 1] - at[i] + S::ROWS - 1) / S::ROWS * tiles;
    }
    if (lane == 31) before[g.groups] = run;
}

// The list of units, in the order that the blocks walk it: groups, of a group the tiles, of a tile the spans (which share its weights).
// `before`: shared memory, units in front of every group; `at`: where its pairs begin. Without offsets there is one group of `rows`.
template <class S>
struct Units {
    const Args& g;
    const int *before, *at;
    int total;
    int e = 0;                            // the group of the unit that was asked for last (units are asked for in ascending order)

    __device__ __forceinline__ Units(const Args& g_, const int* before_, const int* at_) : g(g_), before(before_), at(at_) {
        total = !S::ONE || g.offsets ? before[g.groups] : (g.tiles + S::TILES - 1) / S::TILES * g.spans;
    }
    // the whole warp calls it
    __device__ __forceinline__ Unit operator()(int u) {
        if (S::ONE && !g.offsets) {
            const int t = u / g.spans, first = (u - t * g.spans) * g.span;
            return {0, t * S::TILES, first, min(g.span, g.rows - first), g.span};
        }
        const int lane = threadIdx.x & 31;
        for (;;) {                    // (before[groups] = total > u: it ends)
            const int i = e + 1 + lane;
            const unsigned behind = __ballot_sync(0xffffffffu, i <= g.groups && before[i] <= u);
            e += __popc(behind);
            if (behind != 0xffffffffu) break;
        }
        const int first = at[e], count = at[e + 1] - first, r = u - before[e];
        const int spans = (count + S::ROWS - 1) / S::ROWS, width = ((count + spans - 1) / spans + 15) & ~15, s = r % spans;
        return {e, r / spans * S::TILES, first + s * width, min(width, count - s * width), width};
    }
};
// The same unit in registers that the compiler knows to be the warp's: what the issuing instructions take from the warp's uniform registers is
// otherwise moved there piece by piece (a k block's two copies 390 cycles for 150).
__device__ __forceinline__ Unit uniform(const Unit& u) {
    auto one = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    return {one(u.e), one(u.tile), one(u.first), one(u.here), one(u.width)};
}
// (a cluster's blocks have one unit, and k blocks [lo, lo + n) of it; a block by itself has all of them)
struct Share {
    int unit, step, rank, kb_lo, n_kb;
    __device__ __forceinline__ explicit Share(const Args& g) {
        rank = (int)blockIdx.x % g.blocks, unit = (int)blockIdx.x / g.blocks, step = (int)gridDim.x / g.blocks;
        kb_lo = (int)((long long)g.k_blocks * rank / g.blocks);
        n_kb = (int)((long long)g.k_blocks * (rank + 1) / g.blocks) - kb_lo;
    }
};

// The row that pair p asks with (one that exists, whatever the order says).
__device__ __forceinline__ uint32_t row_of(const Args& g, int p) { return min((uint32_t)(g.order[p] / g.top), (uint32_t)g.rows - 1u); }

// Rows of a unit that lie anywhere, fetched by a warp: this lane's are [16-byte piece lane % 8] of rows r0 + 4 i + lane / 8.
template <class S>
struct Fetch {
    uint32_t piece[S::GATHER_ROWS / 4];   // where the rows begin, in 16-byte pieces
    int rows, under_way = 0, oldest = 0;

    __device__ __forceinline__ void begin(const Args& g, const Unit& unit, int r0) {
        rows = unit.here - r0;
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < S::GATHER_ROWS / 4; ++i) {
            const int r = 4 * i + (lane >> 3);
            if (r < rows) piece[i] = row_of(g, unit.first + r0 + r) * (uint32_t)g.row_step;
        }
    }
    // k block kb into stage s (rows r0 on)
    __device__ __forceinline__ void ask(const Args& g, const Ring<S>& ring, int s, int r0, int kb) {
        const int lane = threadIdx.x & 31, c = lane & 7;
        const int left = min(16, max(0, g.row_bytes - (kb * 128 + c * 16)));          // (behind a row's end: zeros)
        const uint32_t dst = ring.rows(s) + (uint32_t)(r0 + (lane >> 3)) * 128u;
        const uint8_t* a = g.a + (left > 0 ? kb * 128 + c * 16 : 0);
#pragma unroll
        for (int i = 0; i < S::GATHER_ROWS / 4; ++i) {
            const int r = 4 * i + (lane >> 3);          // (r0 is a multiple of 8)
            if (r < rows) cp_async_16(dst + 512u * i + (uint32_t)((c ^ (r & 7)) * 16), a + (size_t)piece[i] * 16, left);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ++under_way;
    }
    // the oldest stage that is still under way has come: the MMAs may read it
    template <int LEFT>
    __device__ __forceinline__ void hand_over(const Ring<S>& ring) {
        asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
        fence_async_proxy();               // (written by threads, read by the tensor cores)
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(ring.full(oldest));
        if (++oldest == ring.stages) oldest = 0;
        --under_way;
    }
    __device__ __forceinline__ void asked(const Ring<S>& ring) {
        if (under_way > FETCHED) hand_over<FETCHED>(ring);
    }
    // at the end, in whatever state: nothing is on its way to memory that is somebody else's next
    __device__ __forceinline__ void end(const Ring<S>& ring, bool ok) {
        if (!ok) asm volatile("cp.async.wait_all;" ::: "memory");
        else
            while (under_way > 0) hand_over<0>(ring);
    }
};

// ---- the copying warps. Returns whether every wait was met; `issued`: k blocks whose copies are under way or done. ----
template <class S, class Fail>
__device__ __forceinline__ bool produce(const CUtensorMap* map_a, const Args& g, const Ring<S>& ring, Units<S>& units, const Share& share, volatile int* abort_flag,
                                        unsigned long long limit, int& issued, Fail fail) {
    bool ok = true, waited = false;
    int s = 0;
    uint32_t parity = 1;                                   // (the first lap finds every stage free)
    [[maybe_unused]] Fetch<S> fetch;
    for (int u = share.unit; u < units.total && ok; u += share.step) {
        const Unit unit = uniform(units(u));
        const bool both = S::TILES == 2 && unit.tile + 1 < g.tiles;
        const uint8_t* w = g.w + ((size_t)((size_t)unit.e * g.tiles + unit.tile) * g.k_blocks + share.kb_lo) * TILE_BYTES;
        const size_t next_tile = (size_t)g.k_blocks * TILE_BYTES;
        const uint32_t bytes = (both ? 2u : 1u) * TILE_BYTES + (g.order ? 0u : (uint32_t)((unit.width + g.box - 1) / g.box * g.box) * 128u);
        auto weights = [&](int s_) {
            mbar_expect_tx(ring.full(s_), bytes);
            bulk_copy(ring.stage(s_), w, TILE_BYTES, ring.full(s_));
            if (both) bulk_copy(ring.stage(s_) + TILE_BYTES, w + next_tile, TILE_BYTES, ring.full(s_));
        };
        auto rows = [&](int s_, int kb) {
            tma_load_2d(ring.rows(s_), map_a, kb * 128, unit.first, ring.full(s_));
            for (int t = g.box; t < unit.width; t += g.box) tma_load_2d(ring.rows(s_) + t * 128, map_a, kb * 128, unit.first + t, ring.full(s_));
        };
        // The first weights are asked for before anything that has to be waited for: of one group in front of the wait for the kernel in front (they are nobody's
        // output), of groups in front of where their rows are.
        int i = 0;
        if (!waited) {
            const int early = min(ring.stages, share.n_kb);
            for (; i < early; ++i, w += TILE_BYTES)
                if (elect_one()) weights(i);
            __syncwarp();
            pdl_wait();
            pdl_trigger();
            waited = true;
            if (S::GATHER == 0 && g.order) fetch.begin(g, unit, 0);
            for (i = 0; i < early; ++i) {
                if (g.order) {
                    if constexpr (S::GATHER == 0) {
                        fetch.ask(g, ring, i, 0, share.kb_lo + i);
                        fetch.asked(ring);
                    }
                } else if (elect_one()) rows(i, share.kb_lo + i);
                __syncwarp();
            }
            issued = early;
            s = early == ring.stages ? 0 : early, parity = early == ring.stages ? 0u : 1u;
        } else if (S::GATHER == 0 && g.order) {
            fetch.begin(g, unit, 0);
        }
        for (; i < share.n_kb; ++i, w += TILE_BYTES) {
            if (!warp_wait(ring.empty(s), parity, abort_flag, 2 * limit)) { ok = false; break; }
            const int kb = share.kb_lo + i;
            if (elect_one()) {
                weights(s);
                if (!g.order) rows(s, kb);
            }
            __syncwarp();
            if constexpr (S::GATHER == 0)
                if (g.order) {
                    fetch.ask(g, ring, s, 0, kb);
                    fetch.asked(ring);
                }
            ++issued;
            if (++s == ring.stages) { s = 0; parity ^= 1u; }
        }
    }
    if (!waited) {
        pdl_wait();
        pdl_trigger();
    }
    if constexpr (S::GATHER == 0)
        if (g.order) fetch.end(ring, ok);
    // (the last lap's releases have arrived too before the block may leave: none is on its way to memory that is somebody else's by then)
    for (int j = max(0, issued - ring.stages); ok && j < issued; ++j)
        ok = warp_wait(ring.empty(j % ring.stages), (uint32_t)(j / ring.stages) & 1u, abort_flag, 2 * limit);
    if (!ok && (threadIdx.x & 31) == 0) fail();
    return ok;
}
// (a warp that fetches rows and nothing else: rows from r0 on)
template <class S, class Fail>
__device__ __forceinline__ bool fetch_rows(const Args& g, const Ring<S>& ring, Units<S>& units, int r0, volatile int* abort_flag, unsigned long long limit, Fail fail) {
    bool ok = true;
    int s = 0;
    uint32_t parity = 1;
    Fetch<S> fetch;
    pdl_wait();
    for (int u = (int)blockIdx.x; u < units.total && ok; u += (int)gridDim.x) {
        const Unit unit = units(u);
        fetch.begin(g, unit, r0);
        for (int kb = 0; kb < g.k_blocks; ++kb) {
            if (!warp_wait(ring.empty(s), parity, abort_flag, 2 * limit)) { ok = false; break; }
            fetch.ask(g, ring, s, r0, kb);
            fetch.asked(ring);
            if (++s == ring.stages) { s = 0; parity ^= 1u; }
        }
    }
    fetch.end(ring, ok);
    if (!ok && (threadIdx.x & 31) == 0) fail();
    return ok;
}

// ---- the issuing warp: M x N as the kernel has its sides (`rows_are_m`) ----
template <bool FP8, bool ROWS_ARE_M, class S, class Fail>
__device__ __forceinline__ bool multiply(const Args& g, const Ring<S>& ring, Units<S>& units, const Share& share, uint32_t tmem_base, volatile int* abort_flag,
                                         unsigned long long limit, int& issued, Fail fail) {
    bool ok = true;
    const uint64_t desc_w0 = smem_desc_sw128(ring.base), desc_r0 = smem_desc_sw128(ring.rows(0));
    uint64_t desc_w = desc_w0, desc_r = desc_r0;          // (a stage further is an addition to the address field)
    int s = 0, buffer = 0;
    uint32_t parity = 0, taken = 1;                        // (the first lap finds every buffer free)
    pdl_wait();          // (the copies are complete no sooner, and the time that the kernel in front still takes is not this wait's)
    for (int u = share.unit; u < units.total && ok; u += share.step) {
        const Unit unit = uniform(units(u));
        const uint32_t kind = idesc<FP8>(ROWS_ARE_M ? 128 * min(S::TILES, g.tiles - unit.tile) : unit.width);
        for (int i = 0; i < share.n_kb; ++i) {
            const int kb = share.kb_lo + i, at = FP8 ? kb % S::TOGETHER : 0;
            const bool opens = i == 0 || (FP8 && at == 0), closes = i == share.n_kb - 1 || (FP8 && at == S::TOGETHER - 1);
            if (opens && !warp_wait(ring.taken(buffer), taken, abort_flag, 2 * limit)) { ok = false; break; }
            if (!warp_wait(ring.full(s), parity, abort_flag, limit)) { ok = false; break; }
            tcgen05_fence_after();
            if (elect_one()) {
                const uint32_t d = tmem_base + (uint32_t)(buffer * S::COLUMNS + at * (S::COLUMNS / S::TOGETHER));
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint64_t m = (ROWS_ARE_M ? desc_r : desc_w) + 2 * k, n = (ROWS_ARE_M ? desc_w : desc_r) + 2 * k;
                    const uint32_t more = (!FP8 && i > 0) || k > 0;
                    if constexpr (FP8) mma_f8(d, m, n, kind, more);
                    else tcgen05_mma_bf16(d, m, n, kind, more);
                }
                tcgen05_commit(ring.empty(s));
                if (closes) tcgen05_commit(ring.sums(buffer));
            }
            __syncwarp();
            ++issued;
            if (closes)
                if (++buffer == S::BUFFERS) { buffer = 0; taken ^= 1u; }
            desc_w += S::STAGE >> 4;
            desc_r += S::STAGE >> 4;
            if (++s == ring.stages) { s = 0; parity ^= 1u; desc_w = desc_w0; desc_r = desc_r0; }
        }
    }
    if (!ok && (threadIdx.x & 31) == 0) fail();
    return ok;
}

// What both kernels begin with: barriers, tensor memory, the lists. Behind it every warp has its role.
template <class S>
__device__ __forceinline__ uint32_t begin(const Args& g, const Ring<S>& ring, int rank, int* before, int* at, uint32_t* tmem_base_slot, int* abort_word) {
    if (threadIdx.x == 0) {
        for (int s = 0; s < ring.stages; ++s) {
            mbar_init(ring.full(s), 1 + (g.order ? S::GATHER_WARPS : 0));
            mbar_init(ring.empty(s), 1 + (g.starve == STARVE_RELEASE && s == 0));
        }
        for (int b = 0; b < S::BUFFERS; ++b) {
            mbar_init(ring.sums(b), 1);
            mbar_init(ring.taken(b), S::EPILOGUE);
        }
        mbar_init(ring.parts(), 1);
        *abort_word = 0;
        if (g.starve == STARVE_COPY && rank == 0) mbar_expect_more(ring.full(0), 16);
        if (g.starve == STARVE_PARTS) mbar_expect_more(ring.parts(), 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (uniform_warp() == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_base_slot)), "r"((uint32_t)S::TMEM) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (!S::ONE || g.offsets) list_units<S>(g, before, at);
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    return *tmem_base_slot;
}
// ... and end with.
template <class S>
__device__ __forceinline__ bool finish_block(const Ring<S>& ring, bool ok, int issued, uint32_t tmem_base, unsigned long long limit) {
    const int warp = uniform_warp(), stages = ring.stages;
    tcgen05_fence_before();
    const bool gave_up = __syncthreads_or(!ok);
    if (gave_up) {
        // (where no wait ran out these have been waited for: the copies by the MMAs, the MMAs by the epilogue and the producer)
        const unsigned long long began = now_ns();
        if (warp == 0)
            for (int j = max(0, issued - stages); j < issued; ++j) drain(ring.full(j % stages), (uint32_t)(j / stages) & 1u, began, limit);
        if (warp == 1 && issued > 0) drain(ring.empty((issued - 1) % stages), (uint32_t)((issued - 1) / stages) & 1u, began, limit);
        __syncthreads();
    }
    if (warp == 1) {
        tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)S::TMEM) : "memory");
    }
    return gave_up;
}

// ---- results ----

// What 16 pairs x 32 weight rows of a warp have come to, parked in shared memory as [16][32] floats -> out, pairs [lo, hi) of the 16 that begin at
// row p0, 16 bytes a lane where `vec`.
template <bool GLU, bool ADDS, typename Tout>
__device__ __forceinline__ void leave(const Finish& f, Tout* out, const float* park, size_t p0, int lo, int hi, int n0, bool vec, int lane) {
    constexpr int PER = 16 / sizeof(Tout);
    if constexpr (GLU) {
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
            if (ADDS && f.accumulate == EPI_ADD) {
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
            *dst = from_float<Tout>(ADDS && f.accumulate == EPI_ADD ? __fadd_rn(v, to_float(*dst)) : v);
        }
    }
}


template <bool FP8, int NT, bool GLU, typename Tout>
__global__ void __launch_bounds__(Narrow<FP8, NT>::THREADS, 2)
gemm_grouped_narrow_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ Args g, Tout* __restrict__ out) {
    using S = Narrow<FP8, NT>;
    constexpr int MINE = NT / S::SETS, CHUNKS = MINE / 16, CLASSES = FP8 && GLU ? 3 : 1;       // a warp's pairs
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(16) float parks[S::EPILOGUE][16 * 32];
    // both scales' products for four k blocks, twice; of gate and up rows there are three scales of the weight in a tile (NT + 4: in other banks)
    __shared__ __align__(16) float scales[FP8 ? 2 : 1][FP8 ? 4 : 1][CLASSES][FP8 ? NT + 4 : 4];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_word;
    const Share share(g);
    Ring<S> ring;
    ring.base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    ring.stages = g.stages;
    uint8_t* aligned = smem_raw + (ring.base - smem_u32(smem_raw));
    const int blocks = g.blocks, rank = share.rank, n_kb = share.n_kb, kb_lo = share.kb_lo;
    const uint32_t parts_at = (uint32_t)g.stages * S::STAGE, part_bytes = (uint32_t)g.share * 128 * 4;      // [share / 4][128 rows][4 tokens]
    ring.bars = ring.base + parts_at + (blocks > 1 ? (uint32_t)blocks * part_bytes : 0u);
    int* before = reinterpret_cast<int*>(aligned + (ring.parts() + 8 - ring.base));
    int* at = before + g.groups + 1;
    const unsigned long long limit = g.limit_us ? g.limit_us * 1000ull : WAIT_NS;
    volatile int* abort_flag = &abort_word;
    // Who waits for another role of the block waits twice as long as that one does for its copies, so that the code names what is missing.
    auto give_up = [&](int code) {
        atomicCAS(g.error_word, 0, code);
        __threadfence();               // (before anybody follows the flag and has a code of his own)
        *abort_flag = 1;
    };
    const uint32_t tmem_base = begin<S>(g, ring, rank, before, at, &tmem_base_slot, &abort_word);
    if (blocks > 1) cluster_arrive();          // (waited for in front of the first send: every block runs and has its barriers)

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    Units<S> units(g, before, at);
    bool ok = true;
    int issued = 0;
    if (warp == 0) {
        ok = produce<S>(&map_a, g, ring, units, share, abort_flag, limit, issued, [&] { give_up(41); });
        if (blocks > 1) cluster_wait();
    } else if (warp == 1) {
        ok = multiply<FP8, false, S>(g, ring, units, share, tmem_base, abort_flag, limit, issued, [&] { give_up(42); });
        if (blocks > 1) cluster_wait();
    } else {
        // ---------------- epilogue: TMEM lanes 32 * (warp % 4) = weight rows of the tile, columns from `t0` on = this warp's pairs ----------------
        const int quad = warp & 3, t0 = ((warp - S::FIRST) >> 2) * MINE, row = quad * 32 + lane, thread = threadIdx.x - 32 * S::FIRST;
        const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)t0;
        float* park = parks[warp - S::FIRST];
        const bool lines = ((uintptr_t)out & 15u) == 0 && (((size_t)g.f.ldo * sizeof(Tout)) & 15u) == 0;
        float4 sw_next[CLASSES];
        [[maybe_unused]] auto ask_weights = [&](const Unit& unit, int kb) {
            const float* sw_row = g.scale_w + (size_t)((size_t)unit.e * g.tiles + unit.tile) * 16 * g.sw_ld + kb;
            sw_next[0] = *reinterpret_cast<const float4*>(sw_row);
            if constexpr (CLASSES == 3) {
                sw_next[1] = *reinterpret_cast<const float4*>(sw_row + g.sw_ld);
                sw_next[2] = *reinterpret_cast<const float4*>(sw_row + 15 * g.sw_ld);
            }
        };
        // (of one group the first weight and its scales are known in front of the wait, and nobody's output)
        if constexpr (FP8)
            if (!g.offsets && thread < NT && share.unit < units.total) ask_weights(units(share.unit), kb_lo & ~3);
        pdl_wait();          // the rows' scales, and what is added into, were written by the kernels before
        int buffer = 0, lap = 0;
        uint32_t parity = 0;
        // (in 8 bits a warp whose wait ran out walks on without work: the block's epilogue warps meet at a barrier)
        for (int u = share.unit; u < units.total && (FP8 || ok); u += share.step) {
            const Unit unit = units(u);
            const int n = unit.tile * 128 + row;
            const float bias = S::ONE && g.f.has_bias && n < g.f.N ? g.f.bias[n] : 0.f;
            const bool vec = lines && n - lane + 32 <= g.f.N;
            // the pairs [lo, hi) of the 16 from t on, parked
            auto finish = [&](int t, int lo, int hi) {
                __syncwarp();
                leave<GLU, S::ONE, Tout>(g.f, out, park, (size_t)(unit.first + t), lo, hi, n - lane, vec, lane);
                __syncwarp();
            };
            auto finished = [&](float v) {
                if constexpr (!S::ONE) return v;
                v = g.f.has_bias ? __fadd_rn(v, bias) : v;
                if (g.f.accumulate == EPI_RELU2) {
                    const float z = v < 0.f ? 0.f : v;              // (what is not a number stays so: a maximum would drop it)
                    v = __fmul_rn(z, z);
                }
                return v;
            };
            if constexpr (FP8) {
                uint64_t sums[MINE / 2];
#pragma unroll
                for (int j = 0; j < MINE / 2; ++j) sums[j] = 0;
                // gate rows' scale, and up rows' in front of and behind the edge of their block of 128: which of them this lane's row has
                const int edge = GLU ? (128 - (((g.f.N >> 1) + unit.tile * 64) & 127)) >> 3 : 0, eight = row >> 3;
                const int kind = GLU && (eight & 1) ? ((eight >> 1) < edge ? 1 : 2) : 0;
                const bool has = thread < unit.here;
                const float* sa_row = g.scale_a + (size_t)(has ? (g.order ? row_of(g, unit.first + thread) : (uint32_t)(unit.first + thread)) : 0u) * g.sa_ld;
                float4 sa_next = make_float4(0.f, 0.f, 0.f, 0.f);
                if (has) sa_next = *reinterpret_cast<const float4*>(sa_row + (kb_lo & ~3));
                if (thread < NT && (g.offsets || u != share.unit)) ask_weights(unit, kb_lo & ~3);
#pragma unroll 1
                for (int kb = kb_lo, end = kb_lo + n_kb; kb < end;) {
                    if (kb == kb_lo || (kb & 3) == 0) {
                        // the scales of four k blocks: asked for four blocks ahead, then shared
                        lap ^= 1;
                        if (thread < NT)
#pragma unroll
                            for (int q = 0; q < CLASSES; ++q) {
                                scales[lap][0][q][thread] = __fmul_rn(sa_next.x, sw_next[q].x);
                                scales[lap][1][q][thread] = __fmul_rn(sa_next.y, sw_next[q].y);
                                scales[lap][2][q][thread] = __fmul_rn(sa_next.z, sw_next[q].z);
                                scales[lap][3][q][thread] = __fmul_rn(sa_next.w, sw_next[q].w);
                            }
                        asm volatile("bar.sync 1, %0;" ::"n"(32 * S::EPILOGUE) : "memory");
                        if (thread < NT && (kb & ~3) + 4 < end) {
                            if (has) sa_next = *reinterpret_cast<const float4*>(sa_row + (kb & ~3) + 4);
                            ask_weights(unit, (kb & ~3) + 4);
                        }
                    }
                    const int first = kb & 1, behind = min((kb | 1) + 1, end) - (kb & ~1);          // of the buffer's two k blocks
                    const float* by = &scales[lap][kb & 2][kind][t0];
                    constexpr int NEXT = CLASSES * (NT + 4);                                          // floats from k block to k block
                    kb = (kb | 1) + 1;
                    if (ok) {
                        ok = __all_sync(0xffffffffu, mbar_wait(ring.sums(buffer), parity, abort_flag, 2 * limit));
                        if (!ok && lane == 0) give_up(43);
                    }
                    if (ok) {
                        tcgen05_fence_after();
                        const uint32_t from = taddr + (uint32_t)(buffer * S::COLUMNS);
                        auto add = [&](const uint32_t* v, const float* s, int c) {
#pragma unroll
                            for (int q = 0; q < 4; ++q) {
                                const ulonglong2 s4 = *reinterpret_cast<const ulonglong2*>(s + 4 * q);
                                asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sums[8 * c + 2 * q]) : "l"(pair_of(v[4 * q], v[4 * q + 1])), "l"(s4.x));
                                asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sums[8 * c + 2 * q + 1]) : "l"(pair_of(v[4 * q + 2], v[4 * q + 3])), "l"(s4.y));
                            }
                        };
                        if (t0 < unit.width) {
                            if constexpr (CHUNKS == 1) {
                                uint32_t v[2][16];
                                if (first == 0) tmem_ld(from, v[0]);
                                if (behind == 2) tmem_ld(from + NT, v[1]);
                                tmem_ld_wait();
                                if (first == 0) add(v[0], by, 0);
                                if (behind == 2) add(v[1], by + NEXT, 0);
                            } else {
#pragma unroll 1
                                for (int j = first; j < behind; ++j) {
                                    uint32_t v[32];
                                    tmem_ld_32x32b_x32(from + j * NT, v);
                                    tmem_ld_wait();
#pragma unroll
                                    for (int c = 0; c < CHUNKS; ++c) add(v + 16 * c, by + j * NEXT + 16 * c, c);
                                }
                            }
                        }
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(ring.taken(buffer));
                    }
                    if (++buffer == S::BUFFERS) { buffer = 0; parity ^= 1u; }
                }
                // the unit's pairs that this warp finishes, 16 at a time: its own, or of a cluster's block its share's
                int t = t0, end = min(t0 + MINE, unit.here), step = 16;
                if (S::CLUSTERS && blocks > 1) {
                    // (one unit a cluster) every block sends what it has of a token to the block that finishes it, itself among them
                    const int tokens = (unit.here + 7) & ~7, part = g.share, lo = rank * part;
                    if (thread == 0) mbar_expect_tx(ring.parts(), (uint32_t)blocks * (uint32_t)max(0, min(part, tokens - lo)) * 512u);
                    cluster_wait();
                    if (ok) {
                        int to = t0 / part, begins = to * part;
                        const uint32_t mine = ring.base + parts_at + (uint32_t)rank * part_bytes + (uint32_t)row * 16;
#pragma unroll
                        for (int q = 0; q < MINE / 4; ++q) {
                            const int tq = t0 + 4 * q;
                            if (tq >= begins + part) ++to, begins += part;
                            if (tq < tokens) {
                                float v[4];
                                halves(sums[2 * q], v[0], v[1]);
                                halves(sums[2 * q + 1], v[2], v[3]);
                                asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                                             ::"r"(in_block(mine + (uint32_t)(tq - begins) * 512u, to)), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])),
                                               "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])), "r"(in_block(ring.parts(), to))
                                             : "memory");
                            }
                        }
                        if (lo < tokens) ok = __all_sync(0xffffffffu, wait_cluster(ring.parts(), 0, abort_flag, 2 * limit));
                        if (!ok && lane == 0) give_up(43);
                    }
                    t = lo + (t0 / MINE) * 16, end = min(lo + part, unit.here), step = 16 * S::SETS;
                }
                if (ok)
#pragma unroll 1
                    for (; t < end; t += step) {
                        if (S::CLUSTERS && blocks > 1) {
                            const uint8_t* parts = aligned + parts_at + (size_t)(t - rank * g.share) * 512 + (size_t)row * 16;
#pragma unroll 1
                            for (int q = 0; q < 4 && t + 4 * q < end; ++q) {
                                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                                for (int p = 0; p < blocks; ++p) {          // (in the blocks' order)
                                    const float4 x = *reinterpret_cast<const float4*>(parts + (size_t)p * part_bytes + q * 2048);
                                    v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
                                }
                                park[(4 * q) * 32 + lane] = finished(v.x);
                                park[(4 * q + 1) * 32 + lane] = finished(v.y);
                                park[(4 * q + 2) * 32 + lane] = finished(v.z);
                                park[(4 * q + 3) * 32 + lane] = finished(v.w);
                            }
                        } else {
#pragma unroll
                            for (int cc = 0; cc < CHUNKS; ++cc)          // (registers are not indexed: one of these runs)
                                if (t == t0 + 16 * cc)
#pragma unroll
                                    for (int q = 0; q < 8; ++q) {
                                        float a, b;
                                        halves(sums[8 * cc + q], a, b);
                                        park[(2 * q) * 32 + lane] = finished(a);
                                        park[(2 * q + 1) * 32 + lane] = finished(b);
                                    }
                        }
                        finish(t, 0, min(16, end - t));
                    }
            } else {
                ok = __all_sync(0xffffffffu, mbar_wait(ring.sums(buffer), parity, abort_flag, 2 * limit));
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t from = taddr + (uint32_t)(buffer * S::COLUMNS);
                const int chunks = min(CHUNKS, (unit.here - t0 + 15) >> 4);
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) {
                    uint32_t v[16];
                    tmem_ld(from + 16 * c, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j) park[j * 32 + lane] = finished(__uint_as_float(v[j]));
                    if (c == chunks - 1) {           // the buffer is another unit's as soon as its last values are read
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(ring.taken(buffer));
                    }
                    finish(t0 + 16 * c, 0, min(16, unit.here - t0 - 16 * c));
                }
                if (chunks <= 0 && lane == 0) mbar_arrive(ring.taken(buffer));
                if (++buffer == S::BUFFERS) { buffer = 0; parity ^= 1u; }
            }
        }
        if (!FP8 && !ok && lane == 0) give_up(43);
    }
    const bool gave_up = finish_block<S>(ring, ok, issued, tmem_base, limit);
    // No block of a cluster leaves before everything sent to it is there: its memory is the next block's at once.
    if (blocks > 1) {
        cluster_arrive();
        cluster_wait();
        if (gave_up) drain(ring.parts(), 0, now_ns(), limit);
    }
}

// ---- many rows to a group: the rows are the M side ----
// A thread of the epilogue has one pair and 64 of the unit's 256 columns: the pair's scale is a register, a tile's scale is one number (of gate and up
// rows three: a block of 128 up rows may end inside the tile), so a k block costs one packed multiply-add for two values.
// Sixteen warps do it: with eight (128 columns each) their way through a k block, one load of tensor memory behind the other, was
// longer than the MMAs' and the copies'.
// A row's 64 bytes of results leave together: a store whose 32 lanes each write 16 bytes of another row costs 32 lines, and what ends a unit stands in
// nobody's shadow (4 us a unit of 128 x 256 that way).
constexpr int WIDE_PARK = 32 * 64;      // bytes of a warp

// N results of this lane's pair into its 64 bytes, from 16-byte piece `first` on: piece c of row r lies at place c ^ (r / 2).
template <typename Tout, int N>
__device__ __forceinline__ void park_row(uint8_t* park, const float (&v)[N], int first, int lane) {
    constexpr int PER = 16 / sizeof(Tout);
#pragma unroll
    for (int c = 0; c < N / PER; ++c) {
        __align__(16) Tout w[PER];
#pragma unroll
        for (int q = 0; q < PER; ++q) w[q] = from_float<Tout>(v[c * PER + q]);
        *reinterpret_cast<uint4*>(park + lane * 64 + (((first + c) ^ (lane >> 1)) & 3) * 16) = *reinterpret_cast<const uint4*>(w);
    }
}
// The warp's 32 rows of 64 bytes -> out, columns from c0 on.
template <bool ADDS, typename Tout>
__device__ __forceinline__ void leave_rows(const Finish& f, Tout* out, uint8_t* park, size_t p0, int rows, int c0, int last, bool vec, int lane) {
    constexpr int PER = 16 / sizeof(Tout), COLS = 4 * PER;
    __syncwarp();
    if (vec && c0 + COLS <= last) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 8 * i + (lane >> 2), c = lane & 3;
            if (r >= rows) continue;
            Tout* dst = out + (p0 + r) * f.ldo + c0 + c * PER;
            uint4 x = *reinterpret_cast<const uint4*>(park + r * 64 + ((c ^ (r >> 1)) & 3) * 16);
            if (ADDS && sizeof(Tout) == 4 && f.accumulate == EPI_ADD) {
                const float4 old = *reinterpret_cast<const float4*>(dst);
                x = make_uint4(__float_as_uint(__fadd_rn(__uint_as_float(x.x), old.x)), __float_as_uint(__fadd_rn(__uint_as_float(x.y), old.y)),
                               __float_as_uint(__fadd_rn(__uint_as_float(x.z), old.z)), __float_as_uint(__fadd_rn(__uint_as_float(x.w), old.w)));
            }
            *reinterpret_cast<uint4*>(dst) = x;
        }
    } else {
        for (int i = lane; i < 32 * COLS; i += 32) {
            const int r = i / COLS, c = i % COLS;
            if (r >= rows || c0 + c >= last) continue;
            Tout* dst = out + (p0 + r) * f.ldo + c0 + c;
            const Tout x = *reinterpret_cast<const Tout*>(park + r * 64 + (((c / PER) ^ (r >> 1)) & 3) * 16 + c % PER * sizeof(Tout));
            *dst = ADDS && sizeof(Tout) == 4 && f.accumulate == EPI_ADD ? from_float<Tout>(__fadd_rn(to_float(x), to_float(*dst))) : x;
        }
    }
}

// CLUSTER: two or four blocks share a unit's k blocks (one unit a cluster). When all have theirs, the rings are idle: each block finishes a part of the unit's
// columns, the others send theirs of it into its ring.
template <bool FP8, bool GLU, bool CLUSTER, typename Tout>
__global__ void __launch_bounds__(Wide<FP8>::THREADS, 1)
gemm_grouped_wide_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ Args g, Tout* __restrict__ out) {
    using S = Wide<FP8>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(16) uint8_t parks[S::EPILOGUE][WIDE_PARK];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_word;
    const Share share(g);
    Ring<S> ring;
    ring.base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    ring.stages = g.stages;
    ring.bars = ring.base + (uint32_t)g.stages * S::STAGE;
    int* before = reinterpret_cast<int*>(smem_raw + (ring.parts() + 8 - smem_u32(smem_raw)));
    int* at = before + g.groups + 1;
    const int n_kb = share.n_kb;
    const unsigned long long limit = g.limit_us ? g.limit_us * 1000ull : WAIT_NS;
    volatile int* abort_flag = &abort_word;
    auto give_up = [&](int code) {
        atomicCAS(g.error_word, 0, code);
        __threadfence();               // (before anybody follows the flag and has a code of his own)
        *abort_flag = 1;
    };
    const uint32_t tmem_base = begin<S>(g, ring, CLUSTER ? share.rank : (int)blockIdx.x, before, at, &tmem_base_slot, &abort_word);

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    Units<S> units(g, before, at);
    bool ok = true;
    int issued = 0;
    if (warp < S::FIRST) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::FEW));
        if (warp == 0) ok = produce<S>(&map_a, g, ring, units, share, abort_flag, limit, issued, [&] { give_up(41); });
        else if (warp == 1) ok = multiply<FP8, true, S>(g, ring, units, share, tmem_base, abort_flag, limit, issued, [&] { give_up(42); });
        else if (g.order) ok = fetch_rows<S>(g, ring, units, (warp - S::GATHER) * S::GATHER_ROWS, abort_flag, limit, [&] { give_up(41); });
        if constexpr (CLUSTER) {
            cluster_arrive();          // (the rings are idle when everybody is here)
            cluster_wait();
        }
    } else {
        // ---------------- epilogue: TMEM lanes 32 * (warp % 4) = the unit's pairs, columns 64 * set on ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::MANY));
        const int quad = warp & 3, set = (warp - S::FIRST) >> 2, half = set >> 1, token = quad * 32 + lane;
        const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(set * 64);
        uint8_t* park = parks[warp - S::FIRST];
        const bool vec = ((uintptr_t)out & 15u) == 0 && (((size_t)g.f.ldo * sizeof(Tout)) & 15u) == 0;
        const int last = GLU ? g.f.N >> 1 : g.f.N;
        pdl_wait();          // the rows' scales, and what is added into, were written by the kernels before
        int buffer = 0;
        uint32_t parity = 0;
        for (int u = share.unit; u < units.total && ok; u += share.step) {
            const Unit unit = units(u);
            const int tile = unit.tile + half, rows = min(32, unit.here - quad * 32), c_set = tile * (GLU ? 64 : 128) + (set & 1) * (GLU ? 32 : 64);
            const bool mine = tile < g.tiles && rows > 0;
            const size_t p0 = (size_t)(unit.first + quad * 32);
            // 16 columns of this lane's pair, the c-th of the warp's, to results
            auto finish = [&](float (&v)[16], int c) {
                constexpr int COLS = 64 / sizeof(Tout);
                if constexpr (GLU) {
                    float eight[8];
                    glu_units<8, true>(g.f.glu, [&](int q) { return v[q]; }, [&](int q) { return v[8 + q]; }, 1.f, eight);
                    constexpr int TIMES = COLS / 8;          // eights of a row's 64 bytes
                    if (c % TIMES == 0) __syncwarp();
                    park_row<Tout>(park, eight, c % TIMES * (4 / TIMES), lane);
                    const int c0 = c_set + c / TIMES * COLS;
                    if (c % TIMES == TIMES - 1 && c0 < last) leave_rows<S::ONE && !GLU, Tout>(g.f, out, park, p0, rows, c0, last, vec, lane);
                } else {
                    const int c16 = c_set + 16 * c;
                    if (S::ONE && g.f.has_bias)
#pragma unroll
                        for (int q = 0; q < 16; ++q) v[q] = c16 + q < last ? __fadd_rn(v[q], g.f.bias[c16 + q]) : 0.f;
                    if (S::ONE && g.f.accumulate == EPI_RELU2)
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            const float z = v[q] < 0.f ? 0.f : v[q];              // (what is not a number stays so: a maximum would drop it)
                            v[q] = __fmul_rn(z, z);
                        }
                    if (S::ONE && sizeof(Tout) == 2 && g.f.accumulate == EPI_ADD && lane < rows) {
                        // (added here, so that the sum is rounded once)
                        const Tout* old = out + (p0 + lane) * g.f.ldo + c16;
#pragma unroll
                        for (int q = 0; q < 16; ++q)
                            if (c16 + q < last) v[q] = __fadd_rn(v[q], to_float(old[q]));
                    }
                    constexpr int TIMES = COLS / 16;
                    if (c % TIMES == 0) __syncwarp();
                    park_row<Tout>(park, v, c % TIMES * (4 / TIMES), lane);
                    const int c0 = c_set + c / TIMES * COLS;
                    if (c % TIMES == TIMES - 1 && c0 < last) leave_rows<S::ONE && !GLU, Tout>(g.f, out, park, p0, rows, c0, last, vec, lane);
                }
            };
            if constexpr (FP8) {
                uint64_t sums[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) sums[j] = 0;
                const bool has = token < unit.here;
                const float* sa_row = g.scale_a + (size_t)(has ? (g.order ? row_of(g, unit.first + token) : (uint32_t)(unit.first + token)) : 0u) * g.sa_ld;
                const float* sw_row = g.scale_w + (size_t)((size_t)unit.e * g.tiles + (tile < g.tiles ? tile : unit.tile)) * 16 * g.sw_ld;
                // of gate and up rows in eights: the gates' scale, and the up rows' in front of and behind the edge of their block of 128
                const int edge = GLU ? ((128 - ((last + tile * 64) & 127)) >> 3) - (set & 1) * 4 : 0;
                constexpr int CLASSES = GLU ? 3 : 1;
                if (lane < CLASSES) sw_row += (lane == 0 ? 0 : lane == 1 ? 1 : 15) * g.sw_ld;
                // The scales of four k blocks, four blocks ahead, in what is the results' place later (two halves: the pairs' [32][4], the weight's [3][4]). (A lane's own
                // loads, one for every k block, took 32 lines each, half of what an SM's cache can do in that time.)
                auto ask = [&](int four, int half_) {
                    const uint32_t to = smem_u32(park) + (uint32_t)half_ * 1024u;
                    cp_async_16(to + (uint32_t)lane * 16u, sa_row + four, has ? 16 : 0);
                    if (lane < CLASSES) cp_async_16(to + 512u + (uint32_t)lane * 16u, sw_row + four, 16);
                };
                int lap = 0;
                const int kb_end = share.kb_lo + n_kb;
                __syncwarp();          // (the unit in front has left)
                ask(share.kb_lo & ~3, 1);
                for (int kb = share.kb_lo; kb < kb_end; ++kb) {
                    if (kb == share.kb_lo || (kb & 3) == 0) {
                        asm volatile("cp.async.wait_all;" ::: "memory");
                        __syncwarp();
                        lap ^= 1;
                        if ((kb & ~3) + 4 < kb_end) ask((kb & ~3) + 4, lap ^ 1);
                    }
                    const float* at_ = reinterpret_cast<const float*>(park) + lap * 256 + (kb & 3);
                    const float sa = at_[lane * 4];
                    uint64_t scale[CLASSES];
#pragma unroll
                    for (int q = 0; q < CLASSES; ++q) {
                        const uint32_t both = __float_as_uint(__fmul_rn(sa, at_[128 + 4 * q]));
                        scale[q] = pair_of(both, both);
                    }
                    ok = __all_sync(0xffffffffu, mbar_wait(ring.sums(buffer), parity, abort_flag, 2 * limit));
                    if (!ok) break;
                    tcgen05_fence_after();
                    const uint32_t from = taddr + (uint32_t)(buffer * S::COLUMNS);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t v[16];
                        tmem_ld(from + 16 * c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const uint64_t by = !GLU || q < 4 ? scale[0] : c < edge ? scale[GLU ? 1 : 0] : scale[GLU ? 2 : 0];
                            asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sums[8 * c + q]) : "l"(pair_of(v[2 * q], v[2 * q + 1])), "l"(by));
                        }
                    }
                    tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(ring.taken(buffer));
                    if (++buffer == S::BUFFERS) { buffer = 0; parity ^= 1u; }
                }
                if (!ok) asm volatile("cp.async.wait_all;" ::: "memory");
                if constexpr (CLUSTER) {
                    // the unit's 16 chunks of 16 columns in order, `per` to a block; a warp's four are one block's
                    const int blocks = g.blocks, rank = share.rank, per = 16 / blocks, owner = set * 4 / per;
                    if (warp == S::FIRST && lane == 0) {
                        const int there = unit.tile + 1 < g.tiles ? per : min(per, max(0, 8 - rank * per));          // (a second tile may be missing)
                        mbar_expect_tx(ring.parts(), (uint32_t)((blocks - 1) * there * unit.here) * 64u);
                    }
                    cluster_arrive();
                    cluster_wait();
                    // [block that sends][chunk][4 columns' place][pair]: 16 bytes
                    if (ok && mine && owner != rank) {
                        const uint32_t to = in_block(ring.base + (uint32_t)((rank - (rank > owner ? 1 : 0)) * per + set * 4 - owner * per) * 8192u + (uint32_t)token * 16u, owner);
                        const uint32_t bar = in_block(ring.parts(), owner);
                        if (lane < rows)
#pragma unroll
                            for (int q = 0; q < 16; ++q) {
                                float v[4];
                                halves(sums[2 * q], v[0], v[1]);
                                halves(sums[2 * q + 1], v[2], v[3]);
                                asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
                                             ::"r"(to + (uint32_t)q * 2048u), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
                                               "r"(__float_as_uint(v[3])), "r"(bar)
                                             : "memory");
                            }
                    }
                    if (ok && mine && owner == rank) ok = __all_sync(0xffffffffu, wait_cluster(ring.parts(), 0, abort_flag, 2 * limit));
                    if (ok && mine && owner == rank) {
                        const uint8_t* parts = smem_raw + (ring.base - smem_u32(smem_raw)) + (size_t)(set * 4 - owner * per) * 8192 + token * 16;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            float v[16];
#pragma unroll
                            for (int q = 0; q < 8; ++q) halves(sums[8 * c + q], v[2 * q], v[2 * q + 1]);
                            for (int p = 0; p < blocks - 1; ++p)
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    const float4 x = *reinterpret_cast<const float4*>(parts + (size_t)p * per * 8192 + (4 * c + q) * 2048);
                                    v[4 * q] += x.x, v[4 * q + 1] += x.y, v[4 * q + 2] += x.z, v[4 * q + 3] += x.w;
                                }
                            finish(v, c);
                        }
                    }
                } else if (ok && mine) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        float v[16];
#pragma unroll
                        for (int q = 0; q < 8; ++q) halves(sums[8 * c + q], v[2 * q], v[2 * q + 1]);
                        finish(v, c);
                    }
                }
            } else {
                ok = __all_sync(0xffffffffu, mbar_wait(ring.sums(buffer), parity, abort_flag, 2 * limit));
                if (!ok) break;
                tcgen05_fence_after();
                const uint32_t from = taddr + (uint32_t)(buffer * S::COLUMNS);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t r[16];
                    tmem_ld(from + 16 * c, r);
                    tmem_ld_wait();
                    if (c == 3) {           // the buffer is another unit's as soon as its last values are read
                        tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(ring.taken(buffer));
                    }
                    float v[16];
#pragma unroll
                    for (int q = 0; q < 16; ++q) v[q] = __uint_as_float(r[q]);
                    if (mine) finish(v, c);
                }
                if (++buffer == S::BUFFERS) { buffer = 0; parity ^= 1u; }
            }
        }
        if (!ok && lane == 0) give_up(43);
    }
    [[maybe_unused]] const bool gave_up = finish_block<S>(ring, ok, issued, tmem_base, limit);
    // No block of a cluster leaves before everything sent to it is there: its memory is the next block's at once.
    if constexpr (CLUSTER) {
        cluster_arrive();
        cluster_wait();
        if (gave_up) drain(ring.parts(), 0, now_ns(), limit);
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------

// Rows of `bytes` bytes, `ld` bytes apart, read in boxes of box_rows x 128 bytes with the 128-byte swizzle.
int rows_map_for(const void* ptr, long long rows, long long bytes, long long ld, int box_rows, CUtensorMap* out) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: the driver does not offer cuTensorMapEncodeTiled");
    const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: cuTensorMapEncodeTiled failed (%d) for [%lld, %lld] bytes, ld %lld", (int)r, rows, bytes, ld);
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
    const BlockRows* rows;
    int pairs, out_dtype;
    void* out;
    cudaStream_t stream;
};

// What a kernel is to the launcher.
struct Kind {
    int rows, tiles;             // of a unit
    size_t stage, fixed, own;    // bytes of a stage, of barriers and alignment, and what the kernel holds by itself
    int tmem, threads;
    int clusters;                // blocks of one at most (0: none)
    bool parts_in_ring;          // what a cluster's blocks send one another lies in their rings, which are idle then (else behind them)
    std::atomic<bool>* allowed;  // [64]: by device, whether the kernel may have an SM's shared memory
};

template <typename Tout>
int launch(void (*kern)(const CUtensorMap, const Args, Tout*), const Kind& kind, const Product& p, const Cut& cut) {
    Args g = p.args;
    const int sms = jllm_device_sm_count(), tiles = (g.tiles + kind.tiles - 1) / kind.tiles;
    if (sms <= 0 || kind.own == 0) return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: the device does not say how many SMs it has, or what the kernel holds");
    // (of groups: every group that has pairs ends one span that is not full)
    const long long spans = g.offsets ? (long long)p.pairs / kind.rows + (g.groups < p.pairs ? g.groups : p.pairs) : ((long long)g.rows + kind.rows - 1) / kind.rows;
    const long long units = spans * tiles;
    JLLM_REQUIRE(units * cut.blocks < BLOCK_MOST, "gemm_grouped: %lld units of work", units);
    g.blocks = cut.blocks;
    // (of the rows of a span, as the units have them)
    const int span = (int)(((g.rows + spans - 1) / spans + 15) / 16 * 16), most_rows = g.rows < span ? g.rows : span;
    g.spans = (int)spans, g.span = span;
    g.share = cut.blocks > 1 ? ((most_rows + 7) / 8 + cut.blocks - 1) / cut.blocks * 8 : 0;
    JLLM_REQUIRE(cut.blocks >= 1 && cut.blocks <= 8 && cut.blocks <= g.k_blocks && (cut.blocks == 1 || (cut.blocks <= kind.clusters && !g.offsets && (!kind.parts_in_ring || 16 % cut.blocks == 0))),
                 "gemm_grouped: no clusters of %d blocks for such a product", cut.blocks);
    // An SM has 228 KB, a block 227 at most; each block's last KB is the system's, `own` what the kernel holds by itself.
    const size_t lists = g.offsets ? 8 * (size_t)(g.groups + 1) : 0, parts = cut.blocks > 1 && !kind.parts_in_ring ? (size_t)cut.blocks * g.share * 512 : 0, fixed = kind.fixed + lists, each = kind.stage + 16;
    const size_t own = kind.own;
    const size_t all = cut.per_sm == 1 ? 227 * 1024 : 113 * 1024;
    JLLM_REQUIRE((cut.per_sm == 1 || cut.per_sm == 2) && kind.tmem * cut.per_sm <= 512 && own + fixed + parts + (FETCHED + 1) * each <= all,
                 "gemm_grouped: %d blocks of such a product on an SM", cut.per_sm);
    int stages = (int)((all - own - fixed - parts) / each);
    if (!g.offsets && cut.blocks == 1) {
        // (no more than a block has k blocks)
        const long long most = (units + (long long)sms * cut.per_sm - 1) / ((long long)sms * cut.per_sm) * g.k_blocks;
        if (stages > most) stages = most < 2 ? 2 : (int)most;
    }
    g.stages = stages;
    // (a span's rows in one copy; of groups some of the next group's come along, of wide ones at most 63)
    g.box = !g.offsets ? span : kind.rows < 64 ? kind.rows : 64;
    CUtensorMap map = {};
    if (!g.order) {          // (fetched rows need none)
        const int rc = rows_map_for(p.rows->data, p.rows->rows, g.row_bytes, p.rows->stride, g.box, &map);
        if (rc != JLLM_OK) return rc;
    }
    // Blocks that wait for one another must not wait for tensor memory that others hold who wait in turn: of a cluster's blocks, which have 256
    // columns at most, no more than two are on an SM (113 KB), nor one beside blocks of another product that together want more than the rest.
    const size_t smem = stages * each + parts + fixed;
    // (what a kernel may have is asked of the driver once per device, and all of it)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: no device");
    if (!kind.allowed[dev].load(std::memory_order_relaxed)) {
        if (cudaFuncSetAttribute((const void*)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(227 * 1024 - own)) != cudaSuccess)
            return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: %zu bytes of shared memory refused", 227 * 1024 - own);
        kind.allowed[dev].store(true, std::memory_order_relaxed);
    }
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
    cudaLaunchKernelEx(&cfg, kern, map, g, static_cast<Tout*>(p.out));
    return jllm_check_launch("gemm_grouped");
}

// What a kernel holds of shared memory by itself; 0 if the driver does not say, or if its threads are launched with fewer registers than `least`.
size_t own_smem(const void* kern, int least = 0) {
    cudaFuncAttributes a{};
    if (cudaFuncGetAttributes(&a, kern) == cudaSuccess) return a.numRegs >= least ? a.sharedSizeBytes : 0;
    cudaGetLastError();
    return 0;
}

template <bool FP8, int NT, bool GLU, typename Tout>
int launch_narrow(const Product& p, const Cut& cut) {
    using S = Narrow<FP8, NT>;
    auto kern = gemm_grouped_narrow_kernel<FP8, NT, GLU, Tout>;
    static const size_t own = own_smem((const void*)kern);
    static std::atomic<bool> allowed[64];
    return launch<Tout>(kern, Kind{S::ROWS, S::TILES, S::STAGE, fixed_smem<S>(), own, S::TMEM, S::THREADS, S::CLUSTERS ? 8 : 0, false, allowed}, p, cut);
}
template <bool FP8, bool GLU, bool CLUSTER, typename Tout>
int launch_wide(const Product& p, const Cut& cut) {
    using S = Wide<FP8>;
    static_assert(3 * 4 * 8192 <= (FETCHED + 1) * S::STAGE, "three blocks' parts of a quarter of the columns, one block's of a half");
    auto kern = gemm_grouped_wide_kernel<FP8, GLU, CLUSTER, Tout>;
    static const size_t own = own_smem((const void*)kern, S::LAUNCHED);          // (what the warps hand over has to be there)
    static std::atomic<bool> allowed[64];
    return launch<Tout>(kern, Kind{S::ROWS, S::TILES, S::STAGE, fixed_smem<S>(), own, S::TMEM, S::THREADS, CLUSTER ? 4 : 0, true, allowed}, p, cut);
}

template <bool FP8, bool GLU, typename Tout>
int launch_cut(const Product& p, const Cut& cut) {
    if (cut.nt == 16 && cut.mt == 1) return launch_narrow<FP8, 16, GLU, Tout>(p, cut);
    if (cut.nt == 32 && cut.mt == 1) return launch_narrow<FP8, 32, GLU, Tout>(p, cut);
    if (cut.nt == 64 && cut.mt == 1) return launch_narrow<FP8, 64, GLU, Tout>(p, cut);
    if (cut.nt == 128 && cut.mt == 2) {
        if constexpr (FP8)
            if (cut.blocks > 1) return launch_wide<FP8, GLU, true, Tout>(p, cut);
        return launch_wide<FP8, GLU, false, Tout>(p, cut);
    }
    return jllm_fail(JLLM_BAD_ARGUMENT, "gemm_grouped: no kernel for spans of %d pairs and %d tiles", cut.nt, cut.mt);
}
template <bool FP8>
int launch_product(const Product& p, const Cut& cut) {
    if (p.out_dtype == JLLM_F32) return p.args.f.glu ? launch_cut<FP8, true, float>(p, cut) : launch_cut<FP8, false, float>(p, cut);
    return p.args.f.glu ? launch_cut<FP8, true, __nv_bfloat16>(p, cut) : launch_cut<FP8, false, __nv_bfloat16>(p, cut);
}

// Clusters of that many blocks that the device runs at a time, `per_sm` blocks an SM; asked once per device.
int resident_clusters(int blocks, int per_sm) {
    static std::atomic<int> known[64][2][9];          // (one more than the answer; who asks first at once with another finds the same)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    std::atomic<int>& answer = known[dev][per_sm - 1][blocks];
    if (const int a = answer.load(std::memory_order_relaxed)) return a - 1;
    using S = Narrow<true, 16>;
    auto kern = gemm_grouped_narrow_kernel<true, 16, false, float>;
    const size_t own = own_smem((const void*)kern), smem = (per_sm == 1 ? 227 * 1024 : 113 * 1024) - own;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (own == 0 || jllm_allow_smem((const void*)kern, smem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    // (the driver counts one block an SM for whatever allocates tensor memory; two run where shared memory has room)
    if (per_sm == 2) {
        const int alone = resident_clusters(blocks, 1);
        if (n < 2 * alone) n = 2 * alone;
    }
    answer.store(n + 1, std::memory_order_relaxed);
    return n;
}

// Counts that put the cuts in order; a count is no time, though it is fitted to microseconds. Fitted to products launched back to back on weights larger
// than L2.
// One weight, e4m3 (4,092 sizes of up to 24 rows, 12,000 of 24 to 2,048, against 128 to 24,576 weight rows of 128 to 12,288 values, up to 20 cuts each; on those that
// the fit has not seen what is chosen is 1.6% slower than the best cut of each size in the geometric mean, 11% at the 95th percentile): a block's k blocks, alone on
// its SM or beside another one, each longer the more SMs take in at once; what a unit costs beside them; sending.
struct Narrowly {
    int nt;
    double start, alone, alone_all, beside, beside_all, unit, send, block, token;
};
constexpr Narrowly NARROW[3] = {{16, 2.57, 0.185, 0.060, 0.167, 0.385, 1.34, 0.711, 0.0352, 0.0579},
                                {32, 2.38, 0.186, 0.113, 0.392, 0.103, 1.65, 0.708, 0.0839, 0.0381},
                                {64, 1.40, 0.329, 0.0721, 0.550, 0.0641, 2.61, 0.0, 0.0, 0.0}};
double narrow_count(const Narrowly& c, int blocks, int rows, int tiles, int k_blocks, int sms) {
    const int one = resident_clusters(blocks, 1), two = resident_clusters(blocks, 2), spans = (rows + c.nt - 1) / c.nt;
    if (blocks > k_blocks || one < 1 || two < 1) return 1e30;
    const long long units = (long long)spans * tiles, all = units * blocks;
    const double each = (k_blocks + blocks - 1) / blocks;
    double run = units <= one ? each * (c.alone + c.alone_all * all / sms) + c.unit
                              : (double)((units + two - 1) / two) * (each * (c.beside + c.beside_all * (all < 2 * sms ? all / (2.0 * sms) : 1.0)) + c.unit);
    if (blocks > 1) run += c.send + c.block * blocks + c.token * ((rows + spans - 1) / spans) * (1.0 - 1.0 / blocks);
    const double read = (double)tiles * TILE_BYTES * k_blocks / 6e6;
    return c.start + (run > read ? run : read);
}
double wide_count(int blocks, int rows, int tiles, int k_blocks, int sms) {
    const int one = resident_clusters(blocks, 1);
    if (blocks > k_blocks || one < 1) return 1e30;
    const long long units = (long long)((tiles + 1) / 2) * ((rows + 127) / 128), rounds = (units + one - 1) / one;
    const double busy = units < one ? (double)units * blocks / sms : 1.0, each = (k_blocks + blocks - 1) / blocks;
    const double run = rounds * (each * (0.455 + 0.124 * busy) + 4.28 + (blocks > 1 ? 5.3 + 0.234 * blocks : 0.0)), read = (double)tiles * TILE_BYTES * k_blocks / 6e6;
    return 1.12 + (run > read ? run : read);
}
// Groups (11,092 sizes: 1 to 2,048 rows of 1 to 8 choices among 4 to 128 groups, 128 to 4,096 weight rows of as many values; 1 to 2% on those that the fit has not seen; by
// the mean of a group's pairs alone 7%): the host knows neither which groups are asked nor how often, so both are reckoned from even choices, half a span more than the pairs fill.
struct Grouping {
    double start, k_block, unit, row;
};
constexpr int SPANS[4] = {16, 32, 64, 128};
constexpr Grouping GROUPING[2][2][4] = {          // [e4m3][by pair][span]
    {{{4.51, 0.263, 0.031, 0.109}, {5.14, 0.264, 0.069, 0.067}, {4.19, 0.645, 0.961, 0.080}, {8.00, 0.327, 4.21, 0.025}},
     {{3.87, 0.219, 0.023, 0.059}, {3.93, 0.229, 0.051, 0.040}, {4.10, 0.220, 0.022, 0.037}, {7.17, 0.175, 0.02, 0.043}}},
    {{{4.03, 0.323, 0.026, 0.154}, {3.98, 0.320, 1.88, 0.046}, {4.05, 0.836, 4.39, 0.065}, {3.04, 0.516, 7.90, 0.036}},
     {{3.76, 0.305, 0.026, 0.132}, {4.58, 0.321, 0.040, 0.075}, {4.75, 0.313, 0.038, 0.072}, {2.24, 0.389, 6.84, 0.020}}}};

// The cut for a product. (Worked out once per size: the choice is kept.)
Cut choose(bool fp8, const RowGroupsView* groups, bool by_pair, int rows, int tiles, int k_blocks) {
    struct Known {
        MapKey key;
        Cut cut;
    };
    static thread_local Known known[256];          // (a place for every size: another size there takes it)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return {16, 1, 1, 2};
    const MapKey key{nullptr, rows + 1, (long long)tiles << 32 | (unsigned)k_blocks, groups ? (long long)groups->groups << 32 | (unsigned)groups->top : 0,
                     dev << 2 | (int)fp8 << 1 | (int)by_pair};
    Known& place = known[MapKeyHash()(key) % 256];
    if (place.key == key) return place.cut;
    const int sms = jllm_device_sm_count();
    Cut best{16, 1, 1, 2};
    double least = 1e30;
    auto offer = [&](double count, const Cut& cut) {
        if (count < least) least = count, best = cut;
    };
    if (!groups) {
        for (const Narrowly& c : NARROW)
            for (int blocks = 1; blocks <= (c.nt <= 32 ? 8 : 1); ++blocks) offer(narrow_count(c, blocks, rows, tiles, k_blocks, sms), {c.nt, 1, blocks, 2});
        for (int blocks = 1; blocks <= 4; blocks *= 2) offer(wide_count(blocks, rows, tiles, k_blocks, sms), {128, 2, blocks, 1});
    } else {
        const double pairs = (double)groups->rows * groups->top, share = groups->top < groups->groups ? (double)groups->top / groups->groups : 1.0;
        const double asked = groups->groups * (1.0 - pow(1.0 - share, groups->rows)), mean = pairs / (asked > 1.0 ? asked : 1.0);
        for (int i = 0; i < 4; ++i) {
            const Grouping& c = GROUPING[fp8][by_pair][i];
            const int nt = SPANS[i], places = nt == 128 ? sms : 2 * sms;
            const double spans = mean <= 0.5 * nt ? asked : pairs / nt + 0.5 * asked, units = spans * (nt == 128 ? (tiles + 1) / 2 : tiles);
            const double rounds = units < places ? 1.0 : units / places, read = asked * tiles * (double)TILE_BYTES * k_blocks / 6.2e6;
            const double run = rounds * (k_blocks * c.k_block + c.unit + c.row * (mean < nt ? mean : nt));
            offer(c.start + sqrt(sqrt(run * run * run * run + read * read * read * read)), {nt, nt == 128 ? 2 : 1, 1, nt == 128 ? 1 : 2});
        }
    }
    place = {key, best};
    return best;
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

// `rows`: what is multiplied (of e4m3, with the scales), [M, K]; `weight`: the packed weight(s) [N, K]; `groups`: null (one weight of e4m3, out [M, N]) or
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
    JLLM_REQUIRE(fp8 || groups, "gemm_grouped: a product of one weight is built for e4m3 rows and weights");
    JLLM_REQUIRE(groups ? groups->groups == weight->groups && groups->groups >= 1 && groups->groups <= MAX_GROUPS && (by_pair ? pairs : groups->rows) == M
                        : weight->groups == 1,
                 "gemm_grouped: %d weights (1 to %d), %d rows and the groups of another product", weight->groups, MAX_GROUPS, M);
    JLLM_REQUIRE(accumulate >= EPI_STORE && accumulate <= EPI_RELU2 && (!groups || (!accumulate && !bias)), "gemm_grouped: accumulate=%d, groups take neither it nor a bias", accumulate);
    JLLM_REQUIRE((swiglu_word != 0) == (weight->glu != 0) && (!swiglu_word || (N % 16 == 0 && !bias && !accumulate)),
                 "gemm_grouped: a gated unit needs a weight packed for it, no bias and no accumulation (N=%d)", N);
    JLLM_REQUIRE(ldo >= (swiglu_word ? N / 2 : N), "gemm_grouped: ldo=%d < N=%d", ldo, N);
    JLLM_REQUIRE((long long)M * (rows->stride / 16) < (1LL << 32) && rows->stride / 16 <= BLOCK_MOST && (long long)K * bytes <= BLOCK_MOST,
                 "gemm_grouped: rows of %lld bytes in all, %lld apart", (long long)M * rows->stride, rows->stride);
    if (pairs == 0) return JLLM_OK;
    int* error_word = jllm_gemm_error_word();
    if (!error_word) return jllm_fail(JLLM_CUDA_ERROR, "gemm_grouped: no error word");
    const bool gather = groups && !by_pair;
    Product p;
    p.args = Args{static_cast<const uint8_t*>(weight->data), static_cast<const uint8_t*>(rows->data), weight->scale, rows->scale, groups ? groups->offsets : nullptr, gather ? groups->order : nullptr,
                  weight->scale_ld, rows->scale_ld, weight->groups, groups ? groups->top : 1, M, (int)pairs, (N + 127) / 128, weight->k_blocks, 0, 0, K * bytes, (int)(rows->stride / 16),
                  Finish{VecRef{bias, bias_dtype}, (int)(bias != nullptr), ldo, accumulate, N, swiglu_word}, 0, 1, 0, 16, starve.what, starve.limit_us, error_word};
    p.rows = rows, p.pairs = (int)pairs, p.out_dtype = out_dtype, p.out = out, p.stream = stream;
    const Cut cut = cut_code ? cut_of(cut_code) : choose(fp8, groups, by_pair != 0, M, p.args.tiles, weight->k_blocks);
    return fp8 ? launch_product<true>(p, cut) : launch_product<false>(p, cut);
}
