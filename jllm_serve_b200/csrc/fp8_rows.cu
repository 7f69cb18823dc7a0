// Rows in 8-bit floating point (e4m3) with a float32 scale for every 128 neighbouring values of a row: scale = max(m, 2^-100) / 448 with m the
// largest magnitude of the 128, rounded to float32, and q = v / scale rounded to e4m3, half to even (448 is e4m3's largest value, so nothing is
// cut off). 128 values that hold an infinity or a NaN have the scale NaN and zeros, so that what is made of them is NaN and not a wrong number.
//
// The quotient is rounded ONCE. t = v * (1 / scale) is off by less than 2 units in its last place, so rounding t is rounding the quotient wherever t
// is further than that from a tie between two e4m3 values; near a tie (about one value in 10^5 of float32 rows; of bfloat16 rows, whose 8
// bits make exact ties common, one in some hundreds) the sign of v - tie * scale decides, which one fused multiply-add gives exactly enough
// (its product is exact and its result has the sign of the exact difference).
//
// Memory bounds it. 16 lanes have a block of 128 values, 8 neighbouring values a lane, so a maximum is four exchanges and nothing meets beyond a
// half warp; a thread has several blocks' values under way at a time.
#include "common.cuh"
#include "fp8_view.h"

namespace {

constexpr float kTiny = 7.888609052210118e-31f;      // 2^-100
constexpr float kMost = 448.f;
constexpr int THREADS = 256, AT_A_TIME = 4;

// Eight values from p on (`left` of them exist); `vec`: 16-byte accesses are allowed.
__device__ __forceinline__ void load8(float (&v)[8], const float* p, int left, bool vec) {
    if (vec && left >= 8) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? p[j] : 0.f;
    }
}
__device__ __forceinline__ void load8(float (&v)[8], const __nv_bfloat16* p, int left, bool vec) {
    if (vec && left >= 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? __bfloat162float(p[j]) : 0.f;
    }
}

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

// v / scale, moved off a tie between two e4m3 values where the quotient is not one: what rounds half to even then rounds the quotient.
__device__ __forceinline__ float quotient(float v, float scale, float inverse) {
    const float t = v * inverse;
    const uint32_t bits = __float_as_uint(t) & 0x7fffffffu;
    // e4m3 values from 2^-6 on have 3 bits behind the leading one: ties are where the 20 bits below are 0x80000. Smaller values lie 2^-9 apart,
    // ties are the odd multiples of 2^-10.
    float tie;
    if (bits >= 0x3c800000u) {          // 2^-6
        const uint32_t below = bits & 0xfffffu;
        if (below - 0x7fffcu > 8u) return t;
        tie = __uint_as_float((bits & ~0xfffffu) | 0x80000u);
    } else {
        const float steps = __uint_as_float(bits) * 1024.f, odd = 2.f * floorf(0.5f * steps) + 1.f;      // (the tie of this e4m3 step)
        if (fabsf(steps - odd) > 1e-4f) return t;
        tie = odd * 0.0009765625f;
    }
    // |v| against tie * scale
    const float beyond = __fmaf_rn(-tie, scale, fabsf(v));
    const float moved = beyond == 0.f ? tie : __uint_as_float(__float_as_uint(tie) + (beyond > 0.f ? 1 : -1));
    return copysignf(moved, v);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) quantize_fp8_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ q, long long ldq, float* __restrict__ scale,
                                                               int ld_scale, int rows, int cols, int blocks, bool vec) {
    pdl_wait();
    pdl_trigger();
    const int lane16 = threadIdx.x & 15;
    const long long items = (long long)rows * blocks, step = (long long)gridDim.x * (THREADS / 16);
    for (long long item = (long long)blockIdx.x * (THREADS / 16) + (threadIdx.x >> 4);; item += AT_A_TIME * step) {
        // (whole warps go on together: the exchanges below are theirs)
        if (!__any_sync(0xffffffffu, item < items)) return;
        float v[AT_A_TIME][8];
        int row[AT_A_TIME], block[AT_A_TIME], left[AT_A_TIME];
#pragma unroll
        for (int a = 0; a < AT_A_TIME; ++a) {
            const long long mine = item + a * step;
            left[a] = 0;
            row[a] = block[a] = 0;
            if (mine < items) {
                split_item(mine, blocks, row[a], block[a]);
                left[a] = min(8, max(0, cols - block[a] * 128 - lane16 * 8));
            } else {
                row[a] = -1;
            }
            if (left[a] > 0) load8(v[a], x + (size_t)row[a] * ldx + block[a] * 128 + lane16 * 8, left[a], vec);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) v[a][j] = 0.f;
        }
#pragma unroll
        for (int a = 0; a < AT_A_TIME; ++a) {
            uint32_t m = 0;                        // (magnitudes as bits: a NaN is larger than everything and stays)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[a][j]) & 0x7fffffffu);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const bool bad = m >= 0x7f800000u;
            const float s = __fdiv_rn(fmaxf(__uint_as_float(bad ? 0u : m), kTiny), kMost), inverse = __frcp_rn(s);
            if (row[a] < 0) continue;
            if (lane16 == 0) scale[(size_t)row[a] * ld_scale + block[a]] = bad ? __uint_as_float(0x7fc00000u) : s;
            uint32_t lo = 0, hi = 0;
            if (!bad) {
                float t[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = quotient(v[a][j], s, inverse);
                lo = e4m3x2(t[0], t[1]) | e4m3x2(t[2], t[3]) << 16;
                hi = e4m3x2(t[4], t[5]) | e4m3x2(t[6], t[7]) << 16;
            }
            // (rows begin at multiples of 16 bytes and have room up to the next one: what is behind the last value is zero)
            const int at = block[a] * 128 + lane16 * 8;
            if (at < ((cols + 15) & ~15)) *reinterpret_cast<uint2*>(q + (size_t)row[a] * ldq + at) = make_uint2(lo, hi);
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
                                                             long long ldo, int rows, int cols, int eights, bool vec) {
    pdl_wait();
    pdl_trigger();
    const long long items = (long long)rows * eights, step = (long long)gridDim.x * THREADS;
    for (long long item = (long long)blockIdx.x * THREADS + threadIdx.x; item < items; item += AT_A_TIME * step) {
        uint2 w[AT_A_TIME];
        float s[AT_A_TIME];
        int row[AT_A_TIME], at[AT_A_TIME];
#pragma unroll
        for (int a = 0; a < AT_A_TIME; ++a)
            if (item + a * step < items) {
                split_item(item + a * step, eights, row[a], at[a]);
                w[a] = *reinterpret_cast<const uint2*>(q + (size_t)row[a] * ldq + at[a] * 8);
                s[a] = scale[(size_t)row[a] * ld_scale + at[a] / 16];
            }
#pragma unroll
        for (int a = 0; a < AT_A_TIME; ++a)
            if (item + a * step < items) {
                float v[8];
                from_e4m3x2(w[a].x & 0xffffu, v[0], v[1]);
                from_e4m3x2(w[a].x >> 16, v[2], v[3]);
                from_e4m3x2(w[a].y & 0xffffu, v[4], v[5]);
                from_e4m3x2(w[a].y >> 16, v[6], v[7]);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], s[a]);
                store8(out + (size_t)row[a] * ldo + at[a] * 8, v, cols - at[a] * 8, vec);
            }
    }
}

// Blocks of threads for `items` threads' work: as many as the SMs hold, or fewer.
int grid_for(long long items, int per_block) {
    const long long all = (items + per_block - 1) / per_block, most = (long long)jllm_device_sm_count() * 8;
    return (int)(all < most ? all : most > 0 ? most : 1);
}

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
    const int blocks = (out->cols + 127) / 128, size = dtype == JLLM_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)x % 16) == 0 && ldx * size % 16 == 0;
    const dim3 grid(grid_for((long long)out->rows * blocks, THREADS / 16));
    uint8_t* q = static_cast<uint8_t*>(const_cast<void*>(out->data));
    float* scale = const_cast<float*>(out->scale);
    if (dtype == JLLM_F32)
        jllm_launch(quantize_fp8_kernel<float>, grid, dim3(THREADS), 0, stream, LAUNCH_DEPENDENT, static_cast<const float*>(x), ldx, q, out->stride, scale,
                    out->scale_ld, out->rows, out->cols, blocks, vec);
    else
        jllm_launch(quantize_fp8_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, stream, LAUNCH_DEPENDENT, static_cast<const __nv_bfloat16*>(x), ldx, q, out->stride,
                    scale, out->scale_ld, out->rows, out->cols, blocks, vec);
    return jllm_check_launch("quantize_fp8");
}

JLLM_EXPORT int jllm_fp8_values(const BlockRows* rows, void* out, int dtype, long long ldo, cudaStream_t stream) {
    const int rc = check("fp8_values", rows);
    if (rc != JLLM_OK) return rc;
    JLLM_REQUIRE(ldo >= rows->cols, "fp8_values: rows of %d values, %lld apart", rows->cols, ldo);
    if (rows->rows == 0) return JLLM_OK;
    const int eights = (rows->cols + 7) / 8, size = dtype == JLLM_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)out % 16) == 0 && ldo * size % 16 == 0;
    const dim3 grid(grid_for((long long)rows->rows * eights, THREADS));
    const uint8_t* q = static_cast<const uint8_t*>(rows->data);
    if (dtype == JLLM_F32)
        jllm_launch(fp8_values_kernel<float>, grid, dim3(THREADS), 0, stream, LAUNCH_DEPENDENT, q, rows->stride, rows->scale, rows->scale_ld, static_cast<float*>(out), ldo,
                    rows->rows, rows->cols, eights, vec);
    else
        jllm_launch(fp8_values_kernel<__nv_bfloat16>, grid, dim3(THREADS), 0, stream, LAUNCH_DEPENDENT, q, rows->stride, rows->scale, rows->scale_ld,
                    static_cast<__nv_bfloat16*>(out), ldo, rows->rows, rows->cols, eights, vec);
    return jllm_check_launch("fp8_values");
}
