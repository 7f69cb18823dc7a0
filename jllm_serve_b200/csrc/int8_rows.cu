// Rows in 8-bit integers: q[r, j] = rint(v[r, j] * (127 / m_r)), scale[r] = m_r / 127 with m_r = max_j |v[r, j]|, so that v is about
// q * scale. Where the values come from: a part's result as it is (quantize_int8), or the residual's addition and the RMS norm in
// front of a product (add_rmsnorm_int8: t = x + y, v = t root gain, root = 1 / sqrt(mean(t^2) + eps)). Sums, maxima and values are
// float32; the one rounding to fewer bits is the one to 8, half to even.
//
// The norm's q does not need the root: with w = t gain it is rint(w * (127 / max |w|)), and scale = root * max |w| / 127. So the sum of
// squares and the maximum are ONE reduction, a row is read once, kept in registers and rounded behind one meeting of its threads.
//
// What a row cannot say in 8 bits: a row whose largest magnitude is below 2^-100 is zeros with scale 0 (127 / m would leave
// float32; of the norm's results such a row may keep its numbers), a row that holds an infinity or a NaN has the scale NaN and zeros, so that what is made of it is NaN and not a wrong number.
//
// Memory bounds them: 2,048 x 4,096 with bfloat16 added 15.9 us for 92 MB (5.8 TB/s, 0.88 of the measured copy), 2,048 x 12,288 quantised 14.1 us
// for 75 MB (5.4 TB/s), 544 x 4,096 added 5.9 us for 25 MB; of a few rows what shows is a launch, one round trip to memory and the meeting (1.3 to
// 2.2 us). What made them so: one reduction where three passes took 63 us; values rounded by an addition and magnitudes compared as integers
// (the quarter-rate conversions bounded 2,048 x 12,288 at 22 us); the gains under way before the wait (10.5 -> 6.9 us at 544 rows).
//
// A thread takes V chunks of 8 neighbouring values, chunk i of a row being thread i % T's. V and T follow from the row's width alone, so
// a row's sum has one order whatever else is in the batch. Rows of up to 512 values are a warp's each, wider ones a block's, beyond 32,768
// values (16,384 of a norm) a thread's chunks are fetched again behind the reduction.
#include "head_rotate.cuh"
#include "int8_view.h"

namespace {

constexpr float kTiny = 7.888609052210118e-31f;      // 2^-100
constexpr int MOST_CHUNKS = 4, MOST_THREADS = 1024;   // what a row's threads hold: 32,768 values; of a norm's, with its gains, half of that
constexpr int NORM_THREADS = 512;

// Magnitudes are compared as the bits of |v|: one integer instruction, and a NaN is larger than everything and stays.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Sum and largest magnitude over the threads of a row: a warp, or (BLOCK) the block's warps. `scratch` holds 64 words.
template <bool BLOCK, bool SUM>
__device__ __forceinline__ void row_reduce(float& sum, uint32_t& m, uint32_t* scratch) {
    if constexpr (SUM) sum = warp_sum(sum);
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (BLOCK) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        __syncthreads();               // (what a reduction in front of this one left has been read)
        if (lane == 0) scratch[warp] = m, scratch[32 + warp] = __float_as_uint(sum);
        __syncthreads();
        m = __reduce_max_sync(0xffffffffu, lane < warps ? scratch[lane] : 0u);
        if constexpr (SUM) sum = warp_sum(lane < warps ? __uint_as_float(scratch[32 + lane]) : 0.f);
    }
}

// Eight values from element i of a row on (`left` of them exist); `vec`: 16-byte accesses are allowed.
__device__ __forceinline__ void load8(float (&v)[8], const float* p, int left, bool vec) {
    if (vec && left >= 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.f;
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8], int left, bool vec) {
    if (vec && left >= 8) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = v[j];
    }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8], int left, bool vec) {
    if (vec && left >= 8) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = __float2bfloat16_rn(v[j]);
    }
}
// Four values rounded to 8 bits. |v * inverse| is at most 127 and a few roundings, so adding 1.5 * 2^23 rounds it to a whole number,
// half to even, which then stands in the lowest byte (a conversion runs at a quarter of the rate and needs its result clamped).
__device__ __forceinline__ uint32_t four_int8(const float* v, float inverse) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(__fadd_rn(__fmul_rn(v[j], inverse), 12582912.f));
    const uint32_t q = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
    return inverse == 0.f ? 0u : q;
}
// ... eight of them stored (q's rows begin at multiples of 16 bytes)
__device__ __forceinline__ void store8(int8_t* p, const float (&v)[8], float inverse, int left) {
    const uint2 w = make_uint2(four_int8(v, inverse), four_int8(v + 4, inverse));
    if (left >= 8) {
        *reinterpret_cast<uint2*>(p) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = (int8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
    }
}

// Eight values as they lie in memory: what a row's threads hold until its scale is known.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p, int left, bool vec) { load8(v, p, left, vec); }
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, magnitude(v[j]));
        return m;
    }
    __device__ __forceinline__ void values(float (&out)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = v[j];
    }
};
template <> struct Raw8<__nv_bfloat16> {
    uint32_t w[4];             // two values each
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int left, bool vec) {
        if (vec && left >= 8) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
            const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = (2 * j < left ? (uint32_t)h[2 * j] : 0u) | (2 * j + 1 < left ? (uint32_t)h[2 * j + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
        for (int j = 1; j < 4; ++j) m = __vmaxu2(m, w[j] & 0x7fff7fffu);
        return max(m << 16, m & 0xffff0000u);
    }
    __device__ __forceinline__ void values(float (&out)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) out[2 * j] = __uint_as_float(w[j] << 16), out[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
};

struct RowScale {
    float scale, inverse;
};
__device__ __forceinline__ RowScale row_scale(uint32_t bits) {
    const float m = __uint_as_float(bits);
    if (!(m < INFINITY)) return {__int_as_float(0x7fffffff), 0.f};
    if (m < kTiny) return {0.f, 0.f};
    return {__fdiv_rn(m, 127.f), __fdiv_rn(127.f, m)};
}

// The row of this thread and its place among the row's threads: (BLOCK) a block's threads have one row, else each warp its own.
template <bool BLOCK> __device__ __forceinline__ int my_row() { return BLOCK ? blockIdx.x : blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); }
template <bool BLOCK> __device__ __forceinline__ int my_place() { return BLOCK ? threadIdx.x : threadIdx.x & 31; }

template <typename T, int V, bool BLOCK>
__global__ void __launch_bounds__(MOST_THREADS) quantize_kernel(const T* __restrict__ x, int ldx, bool vec, int8_t* __restrict__ q, int ldq, float* __restrict__ scale, int rows,
                                int dim) {
    __shared__ uint32_t scratch[64];
    pdl_wait();
    pdl_trigger();
    const int r = my_row<BLOCK>(), at = my_place<BLOCK>() * 8, step = (BLOCK ? blockDim.x : 32) * 8;
    if (r >= rows) return;
    const T* src = x + (size_t)r * ldx;
    int8_t* dst = q + (size_t)r * ldq;
    constexpr bool HELD = V <= MOST_CHUNKS;
    Raw8<T> raw[HELD ? V : 1];
    float unused = 0.f, v[8];
    uint32_t m = 0;
    if constexpr (HELD) {
#pragma unroll
        for (int c = 0; c < V; ++c)
            if (at + c * step < dim) raw[c].load(src + at + c * step, dim - at - c * step, vec);
#pragma unroll
        for (int c = 0; c < V; ++c)
            if (at + c * step < dim) m = max(m, raw[c].largest());
    } else {
        for (int i = at; i < dim; i += step) {
            raw[0].load(src + i, dim - i, vec);
            m = max(m, raw[0].largest());
        }
    }
    row_reduce<BLOCK, false>(unused, m, scratch);
    const RowScale s = row_scale(m);
    if constexpr (HELD) {
#pragma unroll
        for (int c = 0; c < V; ++c)
            if (at + c * step < dim) {
                raw[c].values(v);
                store8(dst + at + c * step, v, s.inverse, dim - at - c * step);
            }
    } else {
        for (int i = at; i < dim; i += step) {
            raw[0].load(src + i, dim - i, vec);
            raw[0].values(v);
            store8(dst + i, v, s.inverse, dim - i);
        }
    }
    if (at == 0) scale[r] = s.scale;
}

struct NormArgs {
    const float* x;
    const void* y;
    float* total;           // may be x
    const void* gain;
    int8_t* q;
    float* scale;
    int ldx, ldy, ldt, ldq, rows, dim;
    float eps;
    bool x_vec, y_vec, t_vec, g_vec;
};

// A row whose squares or products left float32, or vanished in it, or that is zeros or not numbers, in two more passes. First the largest
// magnitudes of t and of w = t gain, which 64 bits hold exactly whatever the two are (of w the upper half: its exponent is what is wanted, and
// an infinity or a NaN shows); then sum and maximum of both, divided by the powers of two that they lie at. A thread reads what it has left
// itself. (A function of its own: nothing of it costs the other rows a register.)
template <typename Tg, bool BLOCK>
__device__ __noinline__ void norm_beyond_float32(const NormArgs& a, int r, uint32_t* scratch) {
    const int at = my_place<BLOCK>() * 8, step = (BLOCK ? blockDim.x : 32) * 8, dim = a.dim;
    const float* t_row = a.y ? a.total + (size_t)r * a.ldt : a.x + (size_t)r * a.ldx;
    const bool t_vec = a.y ? a.t_vec : a.x_vec;
    const Tg* gains = static_cast<const Tg*>(a.gain);
    // f(t, gain) of the chunk at i in place of t
    auto chunk = [&](float (&t)[8], int i, auto&& f) {
        float b[8];
        load8(t, t_row + i, dim - i, t_vec);
        Raw8<Tg> g;
        g.load(gains + i, dim - i, a.g_vec);
        g.values(b);
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = f(t[j], b[j]);
    };
    float t[8], unused = 0.f, ss = 0.f;
    uint32_t top_t = 0, top_w = 0, top = 0;
    for (int i = at; i < dim; i += step)
        chunk(t, i, [&](float v, float g) {
            top_t = max(top_t, magnitude(v));
            top_w = max(top_w, (uint32_t)__double2hiint(__dmul_rn((double)v, (double)g)) & 0x7fffffffu);
            return v;
        });
    row_reduce<BLOCK, false>(unused, top_t, scratch);
    row_reduce<BLOCK, false>(unused, top_w, scratch);
    const bool finite = top_t < 0x7f800000u && top_w < 0x7ff00000u;
    // 2^-exponent of a float64's upper half (1 of zero): in 64 bits even the smallest float32 has an exponent of its own
    auto down = [&](uint32_t high) { return high != 0 && finite ? __hiloint2double((int)((2046u - (high >> 20)) << 20), 0) : 1.0; };
    const double ft = down((uint32_t)__double2hiint((double)__uint_as_float(top_t)) & 0x7fffffffu), fw = down(top_w);
    auto scaled_w = [&](float v, float g) { return (float)((double)v * (double)g * fw); };
    for (int i = at; i < dim; i += step)
        chunk(t, i, [&](float v, float g) {
            const float u = (float)((double)v * ft);
            ss = fmaf(u, u, ss);
            top = max(top, magnitude(scaled_w(v, g)));
            return v;
        });
    row_reduce<BLOCK, true>(ss, top, scratch);
    const float m = __uint_as_float(top);
    const double root = 1.0 / sqrt((double)ss / ft / ft / dim + (double)a.eps);
    const double most = root * ((double)m / fw);                     // (NaN where the row is 0 / 0)
    const bool whole = finite && most < 127.0 * 3.4028234e38;        // (the scale is a number of float32)
    const float inverse = whole && most >= (double)kTiny ? __fdiv_rn(127.f, m) : 0.f;
    for (int i = at; i < dim; i += step) {
        chunk(t, i, scaled_w);
        store8(a.q + (size_t)r * a.ldq + i, t, inverse, dim - i);
    }
    if (at == 0) a.scale[r] = !whole ? __int_as_float(0x7fffffff) : (inverse == 0.f ? 0.f : (float)(most / 127.0));
}

template <typename Ty, typename Tg, int V, bool BLOCK>
__global__ void __launch_bounds__(V <= MOST_CHUNKS ? NORM_THREADS : MOST_THREADS) add_rmsnorm_kernel(const __grid_constant__ NormArgs a) {
    __shared__ uint32_t scratch[64];
    const int r = my_row<BLOCK>(), at = my_place<BLOCK>() * 8, step = (BLOCK ? blockDim.x : 32) * 8, dim = a.dim;
    constexpr bool HELD = V <= MOST_CHUNKS;
    const Tg* gains = static_cast<const Tg*>(a.gain);
    // The gains are nobody's output: they are on their way while the kernel in front ends. (Four chunks of them, held beside the rest,
    // leave too few blocks an SM: 2,048 x 12,288 took 39 us, with the gains asked for chunk by chunk 25.)
    constexpr bool GAINS_HELD = V <= 2;
    Raw8<Tg> gain[GAINS_HELD ? V : 1];
    if constexpr (GAINS_HELD) {
#pragma unroll
        for (int c = 0; c < V; ++c)
            if (at + c * step < dim) gain[c].load(gains + at + c * step, dim - at - c * step, a.g_vec);
    }
    pdl_wait();
    pdl_trigger();
    if (r >= a.rows) return;
    const float* x = a.x + (size_t)r * a.ldx;
    const Ty* y = a.y ? static_cast<const Ty*>(a.y) + (size_t)r * a.ldy : nullptr;
    float* total = a.y ? a.total + (size_t)r * a.ldt : nullptr;
    int8_t* dst = a.q + (size_t)r * a.ldq;
    float ss = 0.f;
    uint32_t top = 0;
    // the chunk at i: t = x + y, left in `total`; t becomes w = t gain
    auto take = [&](float (&t)[8], const Raw8<Ty>& other, const Raw8<Tg>& gain, int i) {
        float b[8];
        if (y) {
            other.values(b);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = __fadd_rn(t[j], b[j]);
            store8(total + i, t, dim - i, a.t_vec);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(t[j], t[j], ss);
        gain.values(b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            t[j] = __fmul_rn(t[j], b[j]);
            top = max(top, magnitude(t[j]));
        }
    };
    float w[HELD ? V : 1][8];
    Raw8<Ty> other[HELD ? V : 1];
    if constexpr (HELD) {
#pragma unroll
        for (int c = 0; c < V; ++c)
            if (at + c * step < dim) {
                load8(w[c], x + at + c * step, dim - at - c * step, a.x_vec);
                if (y) other[c].load(y + at + c * step, dim - at - c * step, a.y_vec);
            }
#pragma unroll
        for (int c = 0; c < V; ++c)
            if (at + c * step < dim) {
                if constexpr (GAINS_HELD) {
                    take(w[c], other[c], gain[c], at + c * step);
                } else {
                    gain[0].load(gains + at + c * step, dim - at - c * step, a.g_vec);
                    take(w[c], other[c], gain[0], at + c * step);
                }
            }
    } else {
        for (int i = at; i < dim; i += step) {
            load8(w[0], x + i, dim - i, a.x_vec);
            if (y) other[0].load(y + i, dim - i, a.y_vec);
            gain[0].load(gains + i, dim - i, a.g_vec);
            take(w[0], other[0], gain[0], i);
        }
    }
    row_reduce<BLOCK, true>(ss, top, scratch);
    float m = __uint_as_float(top);
    if (ss > 1e-24f && ss < 1e30f && m >= kTiny && m < 1e20f) {       // (root below 1e17: the scale stays in float32)
        const float inverse = __fdiv_rn(127.f, m);
        if constexpr (HELD) {
#pragma unroll
            for (int c = 0; c < V; ++c)
                if (at + c * step < dim) store8(dst + at + c * step, w[c], inverse, dim - at - c * step);
        } else {
            for (int i = at; i < dim; i += step) {
                // w once more, from what the thread itself has left
                float t[8], b[8];
                load8(t, (y ? total : x) + i, dim - i, y ? a.t_vec : a.x_vec);
                gain[0].load(gains + i, dim - i, a.g_vec);
                gain[0].values(b);
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = __fmul_rn(t[j], b[j]);
                store8(dst + i, t, inverse, dim - i);
            }
        }
        if (at == 0) a.scale[r] = __fmul_rn(rms_scale(ss, dim, a.eps), __fdiv_rn(m, 127.f));
        return;
    }
    norm_beyond_float32<Tg, BLOCK>(a, r, scratch);
}

// Four 8-bit integers as floats: a byte under the exponent of 2^23 (with its sign bit turned: 128 more than it is), less that.
__device__ __forceinline__ void four_floats(float* v, uint32_t q, float s) {
    q ^= 0x80808080u;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(q, 0x4b000000u, 0x7540 + j)), 8388736.f), s);
}

constexpr int VALUE_ROWS = 4;       // rows that a block of the kernel below goes through
template <typename T>
__global__ void __launch_bounds__(256)
values_kernel(const int8_t* __restrict__ q, int ldq, const float* __restrict__ scale, T* __restrict__ out, int ldo, bool vec, int rows, int dim) {
    pdl_wait();
    pdl_trigger();
    const int at = (blockIdx.x * 256 + threadIdx.x) * 8, left = dim - at;
    if (left <= 0) return;
    for (int group = blockIdx.y; group * VALUE_ROWS < rows; group += gridDim.y) {
        uint2 w[VALUE_ROWS];
        float s[VALUE_ROWS];
        const int lo = group * VALUE_ROWS;
#pragma unroll
        for (int i = 0; i < VALUE_ROWS; ++i)
            if (lo + i < rows) {
                const int8_t* src = q + (size_t)(lo + i) * ldq + at;
                s[i] = scale[lo + i];
                if (left >= 8) {
                    w[i] = *reinterpret_cast<const uint2*>(src);
                } else {
                    w[i] = make_uint2(0, 0);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j < left) (j < 4 ? w[i].x : w[i].y) |= (uint32_t)(uint8_t)src[j] << (8 * (j & 3));
                }
            }
#pragma unroll
        for (int i = 0; i < VALUE_ROWS; ++i)
            if (lo + i < rows) {
                float v[8];
                four_floats(v, w[i].x, s[i]);
                four_floats(v + 4, w[i].y, s[i]);
                store8(out + (size_t)(lo + i) * ldo + at, v, left, vec);
            }
    }
}

// A weight [N, K] of neighbouring bytes a row (ld from row to row) as the tiles that the tensor cores read (gemm_int8.cu); `half` > 0: its rows are
// half gate rows, then as many up rows, and come out in blocks of eight of each.
__global__ void __launch_bounds__(256)
pack_kernel(const int8_t* __restrict__ w, long long ld, int N, int K, int half, int k_blocks, bool vec, uint4* __restrict__ out, long long chunks) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < chunks; i += (long long)gridDim.x * blockDim.x) {
        const int r = (int)(i >> 3) & 127, c = (int)(i & 7) ^ (r & 7);
        const long long block = i >> 10;
        const int tile = (int)(block / k_blocks), k = (int)(block % k_blocks) * 128 + c * 16, n = tile * 128 + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (n < N && k < K) {
            const int row = half > 0 ? (n >> 4) * 8 + (n & 7) + (n & 8 ? half : 0) : n;
            const int8_t* src = w + row * ld + k;
            if (vec && k + 16 <= K) {
                v = *reinterpret_cast<const uint4*>(src);
            } else {
                uint32_t word[4] = {};
                for (int j = 0; j < 16 && k + j < K; ++j) word[j >> 2] |= (uint32_t)(uint8_t)src[j] << (8 * (j & 3));
                v = make_uint4(word[0], word[1], word[2], word[3]);
            }
        }
        out[i] = v;
    }
}

// The threads that share a row of `dim` values and the chunks each holds: two where 512 threads are enough, else four.
struct RowCut {
    int threads, chunks;
};
RowCut row_cut(int dim, int most) {
    const int all = (dim + 7) / 8;
    if (all <= 32) return {32, 1};
    if (all <= 64) return {32, 2};
    const int chunks = all <= 1024 ? 2 : MOST_CHUNKS;
    const int threads = ((all + chunks - 1) / chunks + 31) / 32 * 32;
    return threads <= most ? RowCut{threads, chunks} : RowCut{MOST_THREADS, MOST_CHUNKS + 1};
}
constexpr int WARPS = 4;       // rows of a block whose warps have one each

bool vec16(const void* p, int ld, int size) { return (uintptr_t)p % 16 == 0 && (long long)ld * size % 16 == 0; }

// GO(V, BLOCK): the launch for a row's cut
#define JLLM_ROW_CUT(cut)                                                                    \
    if ((cut).threads == 32 && (cut).chunks == 1) JLLM_GO(1, false);                         \
    else if ((cut).threads == 32) JLLM_GO(2, false);                                         \
    else if ((cut).chunks == 2) JLLM_GO(2, true);                                            \
    else if ((cut).chunks == MOST_CHUNKS) JLLM_GO(MOST_CHUNKS, true);                        \
    else JLLM_GO(MOST_CHUNKS + 1, true)

template <typename T>
void launch_quantize(const void* x, int ldx, int8_t* q, int ldq, float* scale, int rows, int dim, cudaStream_t stream) {
    const RowCut cut = row_cut(dim, MOST_THREADS);
    const bool vec = vec16(x, ldx, sizeof(T));
#define JLLM_GO(V, BLOCK)                                                                                                             \
    jllm_launch(quantize_kernel<T, V, BLOCK>, dim3(BLOCK ? rows : (rows + WARPS - 1) / WARPS), dim3(BLOCK ? cut.threads : 32 * WARPS), 0, \
                stream, LAUNCH_DEPENDENT, static_cast<const T*>(x), ldx, vec, q, ldq, scale, rows, dim)
    JLLM_ROW_CUT(cut);
#undef JLLM_GO
}
template <typename Ty, typename Tg>
void launch_norm(const NormArgs& a, cudaStream_t stream) {
    const RowCut cut = row_cut(a.dim, NORM_THREADS);
#define JLLM_GO(V, BLOCK)                                                                                                                  \
    jllm_launch(add_rmsnorm_kernel<Ty, Tg, V, BLOCK>, dim3(BLOCK ? a.rows : (a.rows + WARPS - 1) / WARPS), dim3(BLOCK ? cut.threads : 32 * WARPS), 0, \
                stream, LAUNCH_DEPENDENT, a)
    JLLM_ROW_CUT(cut);
#undef JLLM_GO
}

}  // namespace

// What all three ask of the int8 rows
#define JLLM_REQUIRE_ROWS(name, v)                                                                                                 \
    JLLM_REQUIRE((v).rows >= 0 && (v).cols > 0 && (v).stride >= (v).cols && vec16((v).data, (v).stride, 1) && (v).rows <= INT8_MOST && \
                     (v).cols <= INT8_MOST,                                                                                         \
                 name ": %d int8 rows of %d values begin at multiples of 16 bytes (stride %d)", (v).rows, (v).cols, (v).stride)

// x [rows, cols] float32 or bfloat16 (row stride ldx) -> the int8 rows of `view`.
JLLM_EXPORT int jllm_quantize_int8(const void* x, int x_dtype, int ldx, const Int8View* view, cudaStream_t stream) {
    const Int8View v = *view;
    JLLM_REQUIRE_ROWS("quantize_int8", v);
    JLLM_REQUIRE(ldx >= v.cols, "quantize_int8: ldx=%d for %d values", ldx, v.cols);
    if (v.rows == 0) return JLLM_OK;
    int8_t* q = const_cast<int8_t*>(v.data);
    float* scale = const_cast<float*>(v.scale);
    if (x_dtype == JLLM_F32) launch_quantize<float>(x, ldx, q, v.stride, scale, v.rows, v.cols, stream);
    else launch_quantize<__nv_bfloat16>(x, ldx, q, v.stride, scale, v.rows, v.cols, stream);
    return jllm_check_launch("quantize_int8");
}

// t = x + y (y null: t = x, and `total` is not written), v = t / sqrt(mean(t^2) + eps) * gain as the int8 rows of `view`; x, total
// float32, y float32 or bfloat16; total may be x.
JLLM_EXPORT int jllm_add_rmsnorm_int8(const float* x, int ldx, const void* y, int y_dtype, int ldy, float* total, int ldt, const void* gain,
                                      int gain_dtype, float eps, const Int8View* view, cudaStream_t stream) {
    const Int8View v = *view;
    JLLM_REQUIRE_ROWS("add_rmsnorm_int8", v);
    JLLM_REQUIRE(ldx >= v.cols && (!y || (ldy >= v.cols && ldt >= v.cols && total)), "add_rmsnorm_int8: ldx=%d ldy=%d ldt=%d for %d values", ldx,
                 ldy, ldt, v.cols);
    if (v.rows == 0) return JLLM_OK;
    const NormArgs a{x, y, total, gain, const_cast<int8_t*>(v.data), const_cast<float*>(v.scale), ldx, ldy, ldt, v.stride,
                     v.rows, v.cols, eps, vec16(x, ldx, 4), vec16(y, ldy, y_dtype == JLLM_F32 ? 4 : 2), vec16(total, ldt, 4),
                     (uintptr_t)gain % 16 == 0};
    const bool g32 = gain_dtype == JLLM_F32;
    if (y_dtype == JLLM_F32) g32 ? launch_norm<float, float>(a, stream) : launch_norm<float, __nv_bfloat16>(a, stream);
    else g32 ? launch_norm<__nv_bfloat16, float>(a, stream) : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, stream);
    return jllm_check_launch("add_rmsnorm_int8");
}

// out[r, j] = q[r, j] * scale[r], float32 or bfloat16.
JLLM_EXPORT int jllm_int8_values(const Int8View* view, void* out, int out_dtype, int ldo, cudaStream_t stream) {
    const Int8View v = *view;
    JLLM_REQUIRE_ROWS("int8_values", v);
    JLLM_REQUIRE(ldo >= v.cols, "int8_values: ldo=%d for %d values", ldo, v.cols);
    if (v.rows == 0) return JLLM_OK;
    const int groups = (v.rows + VALUE_ROWS - 1) / VALUE_ROWS;
    const dim3 blocks((v.cols + 2047) / 2048, groups < 65535 ? groups : 65535);
    if (out_dtype == JLLM_F32)
        jllm_launch(values_kernel<float>, blocks, dim3(256), 0, stream, LAUNCH_DEPENDENT, v.data, v.stride, v.scale, (float*)out, ldo,
                    vec16(out, ldo, 4), v.rows, v.cols);
    else
        jllm_launch(values_kernel<__nv_bfloat16>, blocks, dim3(256), 0, stream, LAUNCH_DEPENDENT, v.data, v.stride, v.scale,
                    (__nv_bfloat16*)out, ldo, vec16(out, ldo, 2), v.rows, v.cols);
    return jllm_check_launch("int8_values");
}

// w [N, K] int8 (row stride ld) -> out [ceil(N / 128)][ceil(K / 128)] tiles of 16 KB; glu: gate rows, then up rows (N a multiple of 16).
JLLM_EXPORT int jllm_pack_int8(const int8_t* w, long long ld, int N, int K, int glu, void* out, cudaStream_t stream) {
    JLLM_REQUIRE(N >= 1 && K >= 1 && (ld >= K || N == 1) && (uintptr_t)out % 16 == 0 && (!glu || N % 16 == 0), "pack_int8: N=%d K=%d ld=%lld", N, K, ld);
    const int k_blocks = (K + 127) / 128;
    const long long chunks = (long long)((N + 127) / 128) * k_blocks * 1024;
    const long long blocks = (chunks + 255) / 256, most = (long long)(jllm_device_sm_count() > 0 ? jllm_device_sm_count() : 1) * 32;
    pack_kernel<<<(int)(blocks < most ? blocks : most), 256, 0, stream>>>(w, ld, N, K, glu ? N / 2 : 0, k_blocks,
                                                                          (uintptr_t)w % 16 == 0 && ld % 16 == 0, static_cast<uint4*>(out), chunks);
    return jllm_check_launch("pack_int8");
}
