// Rows in 8-bit integers: q[r, j] = rint(v[r, j] * (127 / m_r)), scale[r] = m_r / 127 with m_r = max_j |v[r, j]|, so that v is about
// q * scale. Where the values come from: a part's result as it is (quantize_int8), or the residual's addition and the RMS norm in
// front of a product (add_rmsnorm_int8: t = x + y, v = t / sqrt(mean(t^2) + eps) * gain). Sums, maxima and values are float32; the one
// rounding to fewer bits is the one to 8, half to even.
//
// What a row cannot say in 8 bits: a row whose largest magnitude is below 2^-100 is zeros with scale 0 (127 / m would leave
// float32), a row that holds an infinity or a NaN has the scale NaN and zeros, so that what is made of it is NaN and not a wrong number.
#include "head_rotate.cuh"

namespace {

constexpr float kTiny = 7.888609052210118e-31f;      // 2^-100

// The larger of two magnitudes; a NaN stays (fmaxf would drop it).
__device__ __forceinline__ float mag_max(float a, float b) { return a >= b || a != a ? a : b; }
__device__ __forceinline__ float block_mag_max(float v, float* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = mag_max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    v = lane < warps ? scratch[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = mag_max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

struct RowScale {
    float scale, inverse;
};
__device__ __forceinline__ RowScale row_scale(float m) {
    if (!(m < INFINITY)) return {__int_as_float(0x7fffffff), 0.f};
    if (m < kTiny) return {0.f, 0.f};
    return {__fdiv_rn(m, 127.f), __fdiv_rn(127.f, m)};
}
__device__ __forceinline__ int to_int8(float v, float inverse) {
    return inverse == 0.f ? 0 : max(-127, min(127, __float2int_rn(__fmul_rn(v, inverse))));
}

// 1 / sqrt(mean of t^2 + eps) from the sum of squares; where that left float32 (or nearly vanished in it) `again(f)` sums (t f)^2.
template <typename Again>
__device__ __forceinline__ float row_root(float ss, int dim, float eps, Again again) {
    if (ss > 1e-24f && ss < 1e30f) return rms_scale(ss, dim, eps);
    const float f = ss > 1.f ? 8.271806125530277e-25f : 1.2089258196146292e+24f;           // 2^-80, 2^80
    return (float)(1.0 / sqrt((double)again(f) / ((double)f * (double)f) / dim + (double)eps));
}

template <typename T>
__global__ void quantize_kernel(const T* __restrict__ x, int ldx, int8_t* __restrict__ q, int ldq, float* __restrict__ scale, int dim) {
    __shared__ float scratch[33];
    pdl_wait();
    pdl_trigger();
    const T* src = x + (size_t)blockIdx.x * ldx;
    float m = 0.f;
    for (int i = threadIdx.x; i < dim; i += blockDim.x) m = mag_max(m, fabsf(to_float(src[i])));
    const RowScale s = row_scale(block_mag_max(m, scratch));
    int8_t* dst = q + (size_t)blockIdx.x * ldq;
    for (int i = threadIdx.x; i < dim; i += blockDim.x) dst[i] = (int8_t)to_int8(to_float(src[i]), s.inverse);
    if (threadIdx.x == 0) scale[blockIdx.x] = s.scale;
}

template <typename Ty>
__global__ void add_rmsnorm_kernel(const float* x, int ldx, const Ty* __restrict__ y, int ldy, float* total /* may be x */,
                                   int ldt, VecRef gain, float eps, int8_t* __restrict__ q, int ldq, float* __restrict__ scale, int dim) {
    __shared__ float scratch[33];
    pdl_wait();
    pdl_trigger();
    const size_t r = blockIdx.x;
    auto sum_of = [&](int i) { return y != nullptr ? __fadd_rn(x[r * ldx + i], to_float(y[r * ldy + i])) : x[r * ldx + i]; };
    float ss = 0.f, m = 0.f;
    for (int i = threadIdx.x; i < dim; i += blockDim.x) {
        const float t = sum_of(i);
        ss = fmaf(t, t, ss);
    }
    const float root = row_root(block_sum(ss, scratch), dim, eps, [&](float f) {
        float again = 0.f;
        for (int i = threadIdx.x; i < dim; i += blockDim.x) {
            const float t = __fmul_rn(sum_of(i), f);
            again = fmaf(t, t, again);
        }
        return block_sum(again, scratch);
    });
    for (int i = threadIdx.x; i < dim; i += blockDim.x) m = mag_max(m, fabsf(__fmul_rn(__fmul_rn(sum_of(i), root), gain[i])));
    const RowScale s = row_scale(block_mag_max(m, scratch));
    for (int i = threadIdx.x; i < dim; i += blockDim.x) {
        const float t = sum_of(i);
        q[r * ldq + i] = (int8_t)to_int8(__fmul_rn(__fmul_rn(t, root), gain[i]), s.inverse);
        if (y != nullptr) total[r * ldt + i] = t;
    }
    if (threadIdx.x == 0) scale[r] = s.scale;
}

template <typename T>
__global__ void values_kernel(const int8_t* __restrict__ q, int ldq, const float* __restrict__ scale, T* __restrict__ out, int ldo, int dim) {
    pdl_wait();
    pdl_trigger();
    const size_t r = blockIdx.x;
    const float s = scale[r];
    for (int i = threadIdx.x; i < dim; i += blockDim.x) out[r * ldo + i] = from_float<T>(__fmul_rn((float)q[r * ldq + i], s));
}

}  // namespace

// x [rows, dim] float32 or bfloat16 (row stride ldx) -> q int8 (row stride ldq), scale [rows].
JLLM_EXPORT int jllm_quantize_int8(const void* x, int x_dtype, int ldx, int8_t* q, int ldq, float* scale, int rows, int dim, cudaStream_t stream) {
    JLLM_REQUIRE(rows >= 0 && dim > 0 && ldx >= dim && ldq >= dim, "quantize_int8: rows=%d dim=%d ldx=%d ldq=%d", rows, dim, ldx, ldq);
    if (rows == 0) return JLLM_OK;
    if (x_dtype == JLLM_F32)
        jllm_launch(quantize_kernel<float>, dim3(rows), dim3(256), 0, stream, LAUNCH_DEPENDENT, (const float*)x, ldx, q, ldq, scale, dim);
    else
        jllm_launch(quantize_kernel<__nv_bfloat16>, dim3(rows), dim3(256), 0, stream, LAUNCH_DEPENDENT, (const __nv_bfloat16*)x, ldx, q, ldq,
                    scale, dim);
    return jllm_check_launch("quantize_int8");
}

// t = x + y (y null: t = x, and `total` is not written), v = t / sqrt(mean(t^2) + eps) * gain as int8 rows; x, total float32, y float32
// or bfloat16; total may be x.
JLLM_EXPORT int jllm_add_rmsnorm_int8(const float* x, int ldx, const void* y, int y_dtype, int ldy, float* total, int ldt, const void* gain,
                                      int gain_dtype, float eps, int8_t* q, int ldq, float* scale, int rows, int dim, cudaStream_t stream) {
    JLLM_REQUIRE(rows >= 0 && dim > 0 && ldx >= dim && ldq >= dim && (!y || (ldy >= dim && ldt >= dim && total)),
                 "add_rmsnorm_int8: rows=%d dim=%d ldx=%d ldy=%d ldt=%d ldq=%d", rows, dim, ldx, ldy, ldt, ldq);
    if (rows == 0) return JLLM_OK;
    const VecRef g{gain, gain_dtype};
    if (y_dtype == JLLM_F32)
        jllm_launch(add_rmsnorm_kernel<float>, dim3(rows), dim3(256), 0, stream, LAUNCH_DEPENDENT, x, ldx, (const float*)y, ldy, total, ldt, g, eps,
                    q, ldq, scale, dim);
    else
        jllm_launch(add_rmsnorm_kernel<__nv_bfloat16>, dim3(rows), dim3(256), 0, stream, LAUNCH_DEPENDENT, x, ldx, (const __nv_bfloat16*)y, ldy,
                    total, ldt, g, eps, q, ldq, scale, dim);
    return jllm_check_launch("add_rmsnorm_int8");
}

// out[r, j] = q[r, j] * scale[r], float32 or bfloat16.
JLLM_EXPORT int jllm_int8_values(const int8_t* q, int ldq, const float* scale, void* out, int out_dtype, int ldo, int rows, int dim,
                                 cudaStream_t stream) {
    JLLM_REQUIRE(rows >= 0 && dim > 0 && ldq >= dim && ldo >= dim, "int8_values: rows=%d dim=%d ldq=%d ldo=%d", rows, dim, ldq, ldo);
    if (rows == 0) return JLLM_OK;
    if (out_dtype == JLLM_F32)
        jllm_launch(values_kernel<float>, dim3(rows), dim3(256), 0, stream, LAUNCH_DEPENDENT, q, ldq, scale, (float*)out, ldo, dim);
    else
        jllm_launch(values_kernel<__nv_bfloat16>, dim3(rows), dim3(256), 0, stream, LAUNCH_DEPENDENT, q, ldq, scale, (__nv_bfloat16*)out, ldo, dim);
    return jllm_check_launch("int8_values");
}
