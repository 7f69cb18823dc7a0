// Rows in 8-bit floating point (e4m3) with a float32 scale for every 128 neighbouring values of a row: scale = max(m, 2^-100) / 448 with m the
// largest magnitude of the 128, rounded to float32, and q = v / scale rounded to e4m3, half to even (448 is e4m3's largest value, so nothing is
// cut off). 128 values that hold an infinity or a NaN have the scale NaN and zeros, so that what is made of them is NaN and not a wrong number.
//
// The quotient v / scale is rounded ONCE, although float32 arithmetic finds it with an error, and a value next to a tie between two e4m3 values could fall to
// the wrong side.
// float32 rows: v ((1 / scale) (1 - 2^-20)) and v ((1 / scale) (1 + 2^-20)) are both rounded to e4m3, and where they agree that is the quotient's value, which
// lies between them. Where they do not (one value in 10^4), the sign of v - tie * scale decides, which one fused multiply-add gives: its product is exact and
// its result has the sign of the exact difference.
// bfloat16 rows: their 8 bits make ties common (some lane of every second warp has one), so nothing branches. With v = a 2^i and m = b 2^j, a and b of 8 bits,
// v 448 / m is a tie T or further than 2^-13 from it (7 a 2^x and T' b are whole numbers), and the quotient is that, shifted by the error that the scale's own
// rounding left: to the same side for all of a block's values, which m - 448 scale tells. So the reciprocal is taken 2^-20 larger, or smaller; or, where the
// scale is exact, the quotient is corrected by its residual, so that a tie is met exactly and falls to the even value.
//
// Memory bounds it. 16 lanes have a block of 128 values, 8 neighbouring values a lane, so a maximum is four exchanges and nothing meets beyond a
// half warp; a thread has several blocks' values under way at a time. 2,048 x 12,288 bfloat16 17.6 us for 75 MB (4.3 TB/s; the same taken back to bfloat16 13.1
// us, 5.8), float32 22.6 us for 126 MB (5.6); 8 x 4,096 1.65 us.
#include "common.cuh"
#include "fp8_view.h"

namespace {

constexpr float kTiny = 7.888609052210118e-31f;      // 2^-100
constexpr float kMost = 448.f;
constexpr int THREADS = 128, AT_A_TIME = 4;      // blocks of a half warp: neighbours in a row

// Eight neighbouring values of a lane, as they are stored.
template <typename T> struct Eight;
template <> struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
    // (`left` of them exist; `vec`: 16-byte accesses are allowed)
    __device__ __forceinline__ void load(const float* p, int left, bool vec) {
        if (vec && left >= 8) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.f;
        }
    }
    // the bits of the largest magnitude of 16 lanes' values (a NaN is larger than everything and stays)
    __device__ __forceinline__ uint32_t most() const {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        return m;
    }
    __device__ __forceinline__ float value(int j) const { return v[j]; }
};
template <> struct Eight<__nv_bfloat16> {
    uint32_t w[4];
    __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int left, bool vec) {
        if (vec && left >= 8) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = (2 * j < left ? q[2 * j] : 0u) | (2 * j + 1 < left ? (uint32_t)q[2 * j + 1] << 16 : 0u);
        }
    }
    __device__ __forceinline__ uint32_t most() const {
        auto two = [](uint32_t bits) {
            __nv_bfloat162 b;
            *reinterpret_cast<uint32_t*>(&b) = bits & 0x7fff7fffu;
            return b;
        };
        __nv_bfloat162 b = __hmax2_nan(__hmax2_nan(two(w[0]), two(w[1])), __hmax2_nan(two(w[2]), two(w[3])));
        uint32_t m = *reinterpret_cast<const uint32_t*>(&b);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
            b = __hmax2_nan(two(m), two(__shfl_xor_sync(0xffffffffu, m, o)));
            m = *reinterpret_cast<const uint32_t*>(&b);
        }
        return max(m << 16, m & 0xffff0000u);
    }
    __device__ __forceinline__ float value(int j) const { return __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16); }
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void from_e4m3x2(uint32_t two, float& lo, float& hi) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.f32.f16 %0, a;\n\tcvt.f32.f16 %1, b;\n\t}" : "=f"(lo), "=f"(hi) : "r"(h));
}

// Which of two neighbouring e4m3 values `lo` and `hi` (bytes of the same sign; the same one twice: that one) v / scale rounds to: |v| against tie * scale,
// the tie between them; from the tie itself to the even one. `a`, `b`: their magnitudes.
__device__ __forceinline__ uint32_t nearer(float v, float scale, uint32_t lo, uint32_t hi, float a, float b) {
    const float beyond = __fmaf_rn(-0.5f * (a + b), scale, fabsf(v));
    const uint32_t less = min(lo, hi), more = max(lo, hi);          // (bytes of a sign are ordered as their magnitudes)
    return beyond > 0.f || (beyond == 0.f && (less & 1u)) ? more : less;
}
__device__ __forceinline__ uint32_t nearer_two(float v0, float v1, float scale, uint32_t lo, uint32_t hi) {
    float a0, a1, b0, b1;
    from_e4m3x2(lo & 0x7f7fu, a0, a1);
    from_e4m3x2(hi & 0x7f7fu, b0, b1);
    return nearer(v0, scale, lo & 0xffu, hi & 0xffu, a0, b0) | nearer(v1, scale, lo >> 8, hi >> 8, a1, b1) << 8;
}

// Eight values over the scale in e4m3, two to a word; `inverse`: 1 / scale to 2^-22; `off`: the largest magnitude less 448 scales.
__device__ __forceinline__ void rounded(const Eight<float>& v, float scale, float inverse, float, uint32_t (&two)[4]) {
    const float below = inverse * (1.f - 9.5367431640625e-7f), above = inverse * (1.f + 9.5367431640625e-7f);      // 2^-20
    uint32_t hi[4], differ = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        two[j] = e4m3x2(v.value(2 * j) * below, v.value(2 * j + 1) * below);
        hi[j] = e4m3x2(v.value(2 * j) * above, v.value(2 * j + 1) * above);
        differ |= two[j] ^ hi[j];
    }
    if (differ)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (two[j] != hi[j]) two[j] = nearer_two(v.value(2 * j), v.value(2 * j + 1), scale, two[j], hi[j]);
}
__device__ __forceinline__ void rounded(const Eight<__nv_bfloat16>& v, float scale, float inverse, float off, uint32_t (&two)[4]) {
    const float first = off == 0.f ? inverse : inverse * (off > 0.f ? 1.f + 9.5367431640625e-7f : 1.f - 9.5367431640625e-7f), then = off == 0.f ? inverse : 0.f;
    auto quotient = [&](float x) {
        const float t = __fmul_rn(x, first);
        return __fmaf_rn(__fmaf_rn(-t, scale, x), then, t);
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) two[j] = e4m3x2(quotient(v.value(2 * j)), quotient(v.value(2 * j + 1)));
}

// m / 448, correctly rounded: the quotient from the reciprocal and one correction by its residual (P. Markstein, IBM J. Res. Dev. 34, 1990); that it is so for this
// divisor has been counted out over all significands.
__device__ __forceinline__ float by_448(float m) {
    const float y = 0.002232142857142857f, q = __fmul_rn(m, y);
    return __fmaf_rn(__fmaf_rn(-kMost, q, m), y, q);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) quantize_fp8_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq, float* __restrict__ scale,
                                                               int ld_scale, int rows, int cols, int blocks, int chunks, int per, bool vec) {
    pdl_wait();
    pdl_trigger();
    const int lane16 = threadIdx.x & 15;
    const long long items = (long long)rows * chunks, step = (long long)gridDim.x * (THREADS / 16);
    for (long long item = (long long)blockIdx.x * (THREADS / 16) + (threadIdx.x >> 4);; item += step) {
        // (whole warps go on together: the exchanges below are theirs)
        if (!__any_sync(0xffffffffu, item < items)) return;
        int row = 0, first = 0;
        split_item(item, chunks, row, first);
        first *= per;
        const int here = item < items ? min(per, blocks - first) : 0;          // blocks of this half warp
        const T* src = x + (size_t)row * ldx + first * 128 + lane16 * 8;
        const int left = cols - first * 128 - lane16 * 8;                      // values from there on
        Eight<T> v[AT_A_TIME];
#pragma unroll
        for (int a = 0; a < AT_A_TIME; ++a) {
            v[a].zero();
            if (a < here && left > 128 * a) v[a].load(src + 128 * a, left - 128 * a, vec);
        }
        uint8_t* dst = q + (size_t)row * ldq + first * 128 + lane16 * 8;
        float* dst_scale = scale + (size_t)row * ld_scale + first;
#pragma unroll
        for (int a = 0; a < AT_A_TIME; ++a) {
            const uint32_t m = v[a].most();
            if (a >= here) continue;
            const bool bad = m >= 0x7f800000u;
            const float most = fmaxf(__uint_as_float(bad ? 0u : m), kTiny), s = by_448(most), inverse = __fdividef(1.f, s);
            if (lane16 == 0) dst_scale[a] = bad ? __uint_as_float(0x7fc00000u) : s;
            const int values = left - 128 * a;
            if (values <= 0) continue;
            uint32_t two[4];
            rounded(v[a], s, inverse, __fmaf_rn(-kMost, s, most), two);
            const uint2 eight = bad ? make_uint2(0u, 0u) : make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
            if (values >= 8) *reinterpret_cast<uint2*>(dst + 128 * a) = eight;
            else
#pragma unroll
                for (int j = 0; j < 7; ++j)          // (what is behind a row's last value is neither written nor, where rows are read, read)
                    if (j < values) dst[128 * a + j] = (uint8_t)((j < 4 ? eight.x : eight.y) >> 8 * (j & 3));
        }
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
        __align__(16) __nv_bfloat16 w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __float2bfloat16_rn(v[j]);
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(w);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = __float2bfloat16_rn(v[j]);
    }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) fp8_values_kernel(const uint8_t* __restrict__ q, long long ldq, const float* __restrict__ scale, int ld_scale, T* __restrict__ out,
                                                             long long ldo, int rows, int cols, int blocks, int chunks, int per, bool vec) {
    pdl_wait();
    pdl_trigger();
    const int lane16 = threadIdx.x & 15;
    const long long items = (long long)rows * chunks, step = (long long)gridDim.x * (THREADS / 16);
    for (long long item = (long long)blockIdx.x * (THREADS / 16) + (threadIdx.x >> 4); item < items; item += step) {
        int row, first;
        split_item(item, chunks, row, first);
        first *= per;
        const int here = min(per, blocks - first), left = cols - first * 128 - lane16 * 8;
        const uint8_t* src = q + (size_t)row * ldq + first * 128 + lane16 * 8;
        T* dst = out + (size_t)row * ldo + first * 128 + lane16 * 8;
        Bytes8 w[AT_A_TIME];
        float s[AT_A_TIME];
#pragma unroll
        for (int a = 0; a < AT_A_TIME; ++a)
            if (a < here && left > 128 * a) {
                w[a] = bytes_of(src + 128 * a, left - 128 * a);
                s[a] = scale[(size_t)row * ld_scale + first + a];
            }
#pragma unroll
        for (int a = 0; a < AT_A_TIME; ++a)
            if (a < here && left > 128 * a) {
                float v[8];
                from_e4m3x2(w[a].lo & 0xffffu, v[0], v[1]);
                from_e4m3x2(w[a].lo >> 16, v[2], v[3]);
                from_e4m3x2(w[a].hi & 0xffffu, v[4], v[5]);
                from_e4m3x2(w[a].hi >> 16, v[6], v[7]);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], s[a]);
                store8(dst + 128 * a, v, left - 128 * a, vec);
            }
    }
}

// Blocks of threads for `items` half warps' work.
int grid_for(long long items) {
    const long long all = (items + THREADS / 16 - 1) / (THREADS / 16);
    return (int)(all < 0x7fffffff ? all : 0x7fffffff);
}

// A row's blocks in equal chunks: of up to AT_A_TIME, or, where that leaves SMs without a half warp, single ones (8 x 4,096 2.1 -> 1.65 us).
struct Chunks {
    int blocks, chunks, per;
    Chunks(int rows, int cols) : blocks((cols + 127) / 128) {
        const int most = (long long)rows * blocks <= 16LL * jllm_device_sm_count() ? 1 : AT_A_TIME;
        chunks = (blocks + most - 1) / most;
        per = (blocks + chunks - 1) / chunks;
    }
};

int check(const char* name, const BlockRows* r) {
    JLLM_REQUIRE((r->scale || r->rows == 0) && r->rows >= 0 && r->rows <= BLOCK_MOST && r->cols >= 1 && r->cols <= BLOCK_MOST && r->stride % 16 == 0 && r->stride >= r->cols &&
                 ((uintptr_t)r->data % 16) == 0 && r->scale_ld >= (r->cols + 127) / 128,
                 "%s: rows of e4m3 values at multiples of 16 bytes, a scale for each 128 (%d x %d, %lld bytes, %d scales a row)", name, r->rows, r->cols, r->stride, r->scale_ld);
    return JLLM_OK;
}

}  // namespace

JLLM_EXPORT int jllm_quantize_fp8(const void* x, int dtype, long long ldx, const BlockRows* out, cudaStream_t stream) {
    const int rc = check("quantize_fp8", out);
    if (rc != JLLM_OK) return rc;
    JLLM_REQUIRE(ldx >= out->cols, "quantize_fp8: rows of %d values, %lld apart", out->cols, ldx);
    if (out->rows == 0) return JLLM_OK;
    const Chunks c(out->rows, out->cols);
    const int size = dtype == JLLM_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)x % 16) == 0 && ldx * size % 16 == 0;
    const dim3 grid(grid_for((long long)out->rows * c.chunks));
    uint8_t* q = static_cast<uint8_t*>(const_cast<void*>(out->data));
    float* scale = const_cast<float*>(out->scale);
    if (dtype == JLLM_F32)
        jllm_launch(quantize_fp8_kernel<float>, grid, dim3(THREADS), 0, stream, LAUNCH_DEPENDENT, static_cast<const float*>(x), ldx, q, out->stride, scale,
                    out->scale_ld, out->rows, out->cols, c.blocks, c.chunks, c.per, vec);
    else
        jllm_launch(quantize_fp8_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, stream, LAUNCH_DEPENDENT, static_cast<const __nv_bfloat16*>(x), ldx, q, out->stride,
                    scale, out->scale_ld, out->rows, out->cols, c.blocks, c.chunks, c.per, vec);
    return jllm_check_launch("quantize_fp8");
}

JLLM_EXPORT int jllm_fp8_values(const BlockRows* rows, void* out, int dtype, long long ldo, cudaStream_t stream) {
    const int rc = check("fp8_values", rows);
    if (rc != JLLM_OK) return rc;
    JLLM_REQUIRE(ldo >= rows->cols, "fp8_values: rows of %d values, %lld apart", rows->cols, ldo);
    if (rows->rows == 0) return JLLM_OK;
    const Chunks c(rows->rows, rows->cols);
    const int size = dtype == JLLM_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)out % 16) == 0 && ldo * size % 16 == 0;
    const dim3 grid(grid_for((long long)rows->rows * c.chunks));
    const uint8_t* q = static_cast<const uint8_t*>(rows->data);
    if (dtype == JLLM_F32)
        jllm_launch(fp8_values_kernel<float>, grid, dim3(THREADS), 0, stream, LAUNCH_DEPENDENT, q, rows->stride, rows->scale, rows->scale_ld, static_cast<float*>(out), ldo,
                    rows->rows, rows->cols, c.blocks, c.chunks, c.per, vec);
    else
        jllm_launch(fp8_values_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, stream, LAUNCH_DEPENDENT, q, rows->stride, rows->scale, rows->scale_ld,
                    static_cast<__nv_bfloat16*>(out), ldo, rows->rows, rows->cols, c.blocks, c.chunks, c.per, vec);
    return jllm_check_launch("fp8_values");
}
