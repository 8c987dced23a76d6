// Matrix-vector products with 4-bit weights and group scales: the entry point b200wmma_gemv_w4.
//   y[r][i] = alpha * sum_k x[r][k] * s[i][k / G] * (q[i][k] - z[i][k / G]) + beta * y[r][i]
#include "attn_common.cuh"

namespace b200wmma
{
    namespace gemv_w4
    {
        using attn::from_f32;
        using attn::to_f32;

        // One warp to an output of one vector, 8 weights (4 bytes) to a lane at a time.
        template <typename T, typename OutT>
        __global__ void __launch_bounds__(256)
            gemv_w4_kernel(uint32_t m, uint32_t n, const uint8_t* a, uint32_t lda, const T* scales, uint32_t ld_scales, const uint8_t* zeros,
                           uint32_t ld_zeros, uint32_t group, const T* x, uint32_t ldx, OutT* y, uint32_t ldy, float alpha, float beta)
        {
            const uint32_t row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
            if(row >= m)
                return;
            x += size_t(blockIdx.y) * ldx;
            float acc = 0.0f;
            for(uint32_t k = lane * 8; k < n; k += 256)
            {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(a + size_t(row) * lda + k / 2);
                const uint32_t g = k / group;
                const int      z = zeros ? (zeros[size_t(row) * ld_zeros + g] & 15) : 0;
                float          s = 0.0f;
                for(int i = 0; i < 8; ++i)
                {
                    int q = (w >> (4 * i)) & 15;
                    q     = zeros ? q - z : (q ^ 8) - 8;
                    s     = fmaf(to_f32(x[k + i]), static_cast<float>(q), s);
                }
                acc = fmaf(s, to_f32(scales[size_t(row) * ld_scales + g]), acc);
            }
            for(int o = 16; o > 0; o >>= 1)
                acc += __shfl_xor_sync(0xFFFFFFFFu, acc, o);
            if(lane == 0)
            {
                OutT* out = y + size_t(blockIdx.y) * ldy + row;
                acc *= alpha;
                if constexpr(sizeof(OutT) == 4)
                    *out = beta != 0.0f ? acc + beta * *out : acc;
                else
                    *out = from_f32<OutT>(beta != 0.0f ? acc + beta * to_f32(*out) : acc);
            }
        }

        template <typename T, typename OutT>
        static int launch(uint32_t m, uint32_t n, uint32_t rows, const uint8_t* a, uint32_t lda, const void* scales, uint32_t ld_scales,
                          const uint8_t* zeros, uint32_t ld_zeros, uint32_t group, const void* x, uint32_t ldx, void* y, uint32_t ldy,
                          float alpha, float beta, cudaStream_t stream)
        {
            gemv_w4_kernel<T, OutT><<<dim3(ceil_div(m, 8u), rows), 256, 0, stream>>>(m, n, a, lda, static_cast<const T*>(scales), ld_scales,
                                                                                    zeros, ld_zeros, group, static_cast<const T*>(x), ldx,
                                                                                    static_cast<OutT*>(y), ldy, alpha, beta);
            B200_CHECK_CUDA(cudaGetLastError());
            return B200WMMA_OK;
        }
    } // namespace gemv_w4
} // namespace b200wmma

extern "C" int b200wmma_gemv_w4(uint32_t m, uint32_t n, uint32_t rows, const uint8_t* a, uint32_t lda_bytes, const void* scales,
                                uint32_t ld_scales, const uint8_t* zeros, uint32_t ld_zeros, uint32_t group, const void* x, uint32_t ldx,
                                void* y, uint32_t ldy, float alpha, float beta, int data_type, int out_type, void* stream)
{
    using namespace b200wmma;
    clear_error();
    B200_REQUIRE(m && n && rows && group, B200WMMA_ERR_INVALID_ARG, "gemv_w4: m, n, rows and group must be non-zero");
    B200_REQUIRE(a && scales && x && y, B200WMMA_ERR_INVALID_ARG, "gemv_w4: a, scales, x and y must be non-null");
    B200_REQUIRE(data_type == B200WMMA_OUT_F16 || data_type == B200WMMA_OUT_BF16, B200WMMA_ERR_INVALID_ARG,
                 "gemv_w4: data_type must be B200WMMA_OUT_F16 or B200WMMA_OUT_BF16");
    B200_REQUIRE(out_type == data_type || out_type == B200WMMA_OUT_F32, B200WMMA_ERR_INVALID_ARG,
                 "gemv_w4: out_type must be data_type or B200WMMA_OUT_F32");
    B200_REQUIRE(n % 32 == 0 && group % 32 == 0, B200WMMA_ERR_UNSUPPORTED, "gemv_w4: n and group must be multiples of 32");
    B200_REQUIRE(m < (1u << 31) && rows < 65536u, B200WMMA_ERR_UNSUPPORTED, "gemv_w4: m must be below 2^31 and rows below 65536");
    const uint32_t groups = (n - 1) / group + 1;
    B200_REQUIRE(lda_bytes >= n / 2 && ldx >= n && ldy >= m && ld_scales >= groups && (!zeros || ld_zeros >= groups),
                 B200WMMA_ERR_INVALID_ARG, "gemv_w4: a leading dimension is smaller than its row");
    B200_REQUIRE(aligned16(a) && lda_bytes % 16 == 0 && aligned16(x) && ldx % 8 == 0, B200WMMA_ERR_ALIGNMENT,
                 "gemv_w4: a, x and their leading dimensions must be multiples of 16 bytes");
    if(int e = require_sm100())
        return e;
    const auto run = [&](auto fn) {
        return fn(m, n, rows, a, lda_bytes, scales, ld_scales, zeros, ld_zeros, group, x, ldx, y, ldy, alpha, beta, as_stream(stream));
    };
    if(data_type == B200WMMA_OUT_F16)
        return out_type == B200WMMA_OUT_F32 ? run(gemv_w4::launch<__half, float>) : run(gemv_w4::launch<__half, __half>);
    return out_type == B200WMMA_OUT_F32 ? run(gemv_w4::launch<__nv_bfloat16, float>) : run(gemv_w4::launch<__nv_bfloat16, __nv_bfloat16>);
}
