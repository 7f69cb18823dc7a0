// out[m, n] (+)= (sum_k qa[m, k] * qw[n, k]) * scale_a[m] * scale_w[n] (+ bias[n]), 8-bit integers with one scale a token and one a
// weight row. The sum is exact in 32-bit integers (k up to 131,071: 131,071 * 128 * 128 < 2^31), so its order does not matter: every
// way of cutting the work gives the same bits, and a row's result does not depend on what else is in the batch.
//
// The weight is PACKED once (ops.pack_int8): tiles of 128 rows x 128 k, each the 16 KB image that the tensor cores read from shared
// memory (rows of 128 bytes, 16-byte chunk c of row r at chunk position c ^ (r & 7)), tile (t, kb) at (t * k_blocks + kb) * 16 KB.
#include "common.cuh"

namespace {

constexpr int BK = 128, TILE_BYTES = 128 * BK;
constexpr int MAX_K = 131071;

// The result from the exact sum, the same operations in the same order in every kernel.
__device__ __forceinline__ float scaled(int sum, float scale_a, float scale_w) { return __fmul_rn(__fmul_rn((float)sum, scale_a), scale_w); }

// 32 weight rows x 32 tokens a block: a lane has a weight row, a warp four tokens.
template <typename Tout>
__global__ void __launch_bounds__(256)
gemm_int8_kernel(const int8_t* __restrict__ a, int lda, const float* __restrict__ scale_a, const int8_t* __restrict__ w,
                 const float* __restrict__ scale_w, int k_blocks, VecRef bias, int has_bias, Tout* __restrict__ out, int ldo, int accumulate,
                 int M, int N, int K, GluArgs swiglu) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, n = blockIdx.x * 32 + lane, m0 = blockIdx.y * 32 + (threadIdx.x >> 5) * 4, row = n & 127;
    if (m0 >= M) return;
    int sum[4] = {};
    const int8_t* wt = w + (size_t)(n >> 7) * k_blocks * TILE_BYTES + row * BK;
    for (int k = 0; k < K; k += 16) {
        const int8_t* p = wt + (size_t)(k / BK) * TILE_BYTES + ((((k % BK) >> 4) ^ (row & 7)) << 4);
        const int4 wv = *reinterpret_cast<const int4*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (m0 + j >= M) break;
            const int8_t* src = a + (size_t)(m0 + j) * lda + k;
            if (k + 16 <= K) {
                const int4 av = *reinterpret_cast<const int4*>(src);
                sum[j] = __dp4a(av.x, wv.x, sum[j]);
                sum[j] = __dp4a(av.y, wv.y, sum[j]);
                sum[j] = __dp4a(av.z, wv.z, sum[j]);
                sum[j] = __dp4a(av.w, wv.w, sum[j]);
            } else {
                for (int i = 0; i < K - k; ++i) sum[j] += (int)src[i] * (int)p[i];
            }
        }
    }
    const float sw = n < N ? scale_w[n] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (m0 + j >= M) break;
        const float v = scaled(sum[j], scale_a[m0 + j], sw);
        if (swiglu) {
            const float up = __shfl_xor_sync(0xffffffffu, v, 8);
            const int unit = (n >> 4) * 8 + (n & 7);
            if ((lane & 8) == 0 && n + 8 < N) {
                float one[1];
                glu_units<1>(swiglu.word_of(unit), [&](int) { return v; }, [&](int) { return up; }, 1.f, one);
                out[(size_t)(m0 + j) * ldo + unit] = from_float<Tout>(one[0]);
            }
        } else if (n < N) {
            float r = epilogue_act(has_bias ? __fadd_rn(v, bias[n]) : v, accumulate);
            Tout* dst = out + (size_t)(m0 + j) * ldo + n;
            if (accumulate == EPI_ADD) r = __fadd_rn(r, to_float(*dst));
            *dst = from_float<Tout>(r);
        }
    }
}

}  // namespace

// a [M, K] int8 (row stride lda, a multiple of 16), w_packed: ops.pack_int8 of the [N, K] weight, out [M, N] (or [M, N / 2] with
// swiglu) float32 or bfloat16.
JLLM_EXPORT int jllm_gemm_int8(const int8_t* a, int lda, const float* scale_a, const int8_t* w_packed, const float* scale_w, int k_blocks,
                               const void* bias, int bias_dtype, void* out, int out_dtype, int ldo, int accumulate, int M, int N, int K,
                               int swiglu_word, cudaStream_t stream) {
    const GluArgs swiglu = glu_args(swiglu_word, nullptr);
    JLLM_REQUIRE(M >= 0 && N >= 1 && K >= 1 && K <= MAX_K, "gemm_int8: M=%d N=%d K=%d (K from 1 to %d)", M, N, K, MAX_K);
    JLLM_REQUIRE(lda >= K && lda % 16 == 0 && ((uintptr_t)a % 16) == 0 && ((uintptr_t)w_packed % 16) == 0,
                 "gemm_int8: rows and weights begin at multiples of 16 bytes (lda=%d, K=%d)", lda, K);
    JLLM_REQUIRE(k_blocks == (K + BK - 1) / BK, "gemm_int8: the packed weight has %d k blocks, K=%d needs %d", k_blocks, K, (K + BK - 1) / BK);
    JLLM_REQUIRE(accumulate >= EPI_STORE && accumulate <= EPI_RELU2, "gemm_int8: accumulate=%d", accumulate);
    JLLM_REQUIRE(ldo >= (swiglu ? N / 2 : N), "gemm_int8: ldo=%d < N=%d", ldo, N);
    JLLM_REQUIRE(!swiglu || (N % 16 == 0 && !bias && !accumulate),
                 "gemm_int8: the SwiGLU epilogue needs N %% 16 == 0, no bias and no accumulation (N=%d)", N);
    if (M == 0) return JLLM_OK;
    const VecRef b{bias, bias_dtype};
    const dim3 grid((N + 31) / 32, (M + 31) / 32);
    JLLM_REQUIRE(grid.y < 65536, "gemm_int8: %d rows", M);
    if (out_dtype == JLLM_F32)
        jllm_launch(gemm_int8_kernel<float>, grid, dim3(256), 0, stream, LAUNCH_DEPENDENT, a, lda, scale_a, w_packed, scale_w, k_blocks, b,
                    (int)(bias != nullptr), (float*)out, ldo, accumulate, M, N, K, swiglu);
    else
        jllm_launch(gemm_int8_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, LAUNCH_DEPENDENT, a, lda, scale_a, w_packed, scale_w, k_blocks, b,
                    (int)(bias != nullptr), (__nv_bfloat16*)out, ldo, accumulate, M, N, K, swiglu);
    return jllm_check_launch("gemm_int8");
}
