// What the attention kernels share: the checked and flattened arguments, and the arithmetic of one score
//   s = cap * tanh(scale * q.k / cap) - slope * |distance|,  masked by causality, prefix and documents.
#pragma once
#include "common.cuh"

#include <atomic>
#include <cuda_bf16.h>
#include <type_traits>

namespace b200wmma
{
    namespace attn
    {
        constexpr uint32_t MAX_DIM = 128;
        constexpr float    LOG2E   = 1.4426950408889634f;
        constexpr float    LN2     = 0.6931471805599453f;

        struct Strides
        {
            int64_t batch, token, head;
        };

        // Kernel parameters of the forward and backward pass.
        struct Params
        {
            uint32_t batch, heads_q, heads_kv, len_q, len_kv, dim;
            int32_t  off; // len_kv - len_q: query i stands at key position i + off
            int32_t  causal;
            float    scale, cap;
            const float*   slopes;
            const int32_t *prefix, *doc_q, *doc_kv;
            Strides        q, k, v, o, dout, dq, dk, dv;
        };

        template <typename T>
        __device__ __forceinline__ float to_f32(T x)
        {
            if constexpr(std::is_same<T, __half>::value)
                return __half2float(x);
            else
                return __bfloat162float(x);
        }
        template <typename T>
        __device__ __forceinline__ T from_f32(float x)
        {
            if constexpr(std::is_same<T, __half>::value)
                return __float2half_rn(x);
            else
                return __float2bfloat16_rn(x);
        }

        // Lets a kernel use this much dynamic shared memory; asked of the driver once per device and kernel (`allowed` is the
        // kernel's own), which saves a launch-bound caller half a microsecond a call.  `bytes` has to be the same in every call of
        // a kernel, the most that any launch of it takes: threads that come here for the first time at once all ask the driver.
        using Allowed = std::atomic<bool>[MAX_DEVICES];
        static int allow_smem(const void* kern, uint32_t bytes, Allowed& allowed)
        {
            std::atomic<bool>& asked = allowed[current_device_slot()];
            if(!asked.load(std::memory_order_acquire))
            {
                B200_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
                asked.store(true, std::memory_order_release);
            }
            return B200WMMA_OK;
        }

        // ---- host side: argument checks -------------------------------------------------------
        static int check_strides(const char* who, const char* name, const void* base, const b200wmma_attn_strides& s,
                                 uint32_t batch, uint32_t tokens, uint32_t heads, Strides* out)
        {
            B200_REQUIRE(base, B200WMMA_ERR_INVALID_ARG, "%s: %s must be non-null", who, name);
            B200_REQUIRE(aligned16(base), B200WMMA_ERR_ALIGNMENT, "%s: %s must be 16-byte aligned", who, name);
            const int64_t  st[3]  = {s.batch, s.token, s.head};
            const uint32_t ext[3] = {batch, tokens, heads};
            static const char* const which[3] = {"batch", "token", "head"};
            int64_t                  v[3];
            for(int i = 0; i < 3; ++i)
            {
                v[i] = ext[i] > 1 ? st[i] : 8;
                B200_REQUIRE(v[i] > 0, B200WMMA_ERR_INVALID_ARG, "%s: the %s stride of %s must be positive", who, which[i], name);
                B200_REQUIRE(v[i] % 8 == 0, B200WMMA_ERR_ALIGNMENT, "%s: the %s stride of %s must be a multiple of 8 elements", who,
                             which[i], name);
                B200_REQUIRE(v[i] < (int64_t(1) << 38), B200WMMA_ERR_UNSUPPORTED, "%s: the %s stride of %s is too large", who,
                             which[i], name);
            }
            *out = {v[0], v[1], v[2]};
            return B200WMMA_OK;
        }
        // The elements that a call writes must not share memory among themselves.  Of three extents, sorted by stride, each
        // stride has to clear what the smaller ones span; rows are `dim` elements.
        static bool disjoint(const Strides& s, uint32_t batch, uint32_t tokens, uint32_t heads, uint32_t dim)
        {
            int64_t  st[3] = {s.batch, s.token, s.head};
            uint32_t n[3]  = {batch, tokens, heads};
            for(int i = 0; i < 3; ++i)
                for(int j = i + 1; j < 3; ++j)
                    if(st[j] < st[i])
                    {
                        const int64_t t = st[i];
                        st[i] = st[j], st[j] = t;
                        const uint32_t u = n[i];
                        n[i] = n[j], n[j] = u;
                    }
            int64_t span = dim;
            for(int i = 0; i < 3; ++i)
            {
                if(n[i] <= 1)
                    continue;
                if(st[i] < span)
                    return false;
                span += st[i] * (int64_t(n[i]) - 1);
            }
            return true;
        }

        static int check_common(const char* who, const b200wmma_attn_args* a)
        {
            B200_REQUIRE(a, B200WMMA_ERR_INVALID_ARG, "%s: args must be non-null", who);
            B200_REQUIRE(a->batch && a->heads_q && a->heads_kv && a->head_dim, B200WMMA_ERR_INVALID_ARG,
                         "%s: batch, heads_q, heads_kv and head_dim must be non-zero", who);
            B200_REQUIRE(a->heads_q % a->heads_kv == 0, B200WMMA_ERR_INVALID_ARG, "%s: heads_q must be a multiple of heads_kv", who);
            B200_REQUIRE(a->head_dim % 8 == 0 && a->head_dim <= MAX_DIM, B200WMMA_ERR_UNSUPPORTED,
                         "%s: head_dim must be a multiple of 8, at most %u", who, MAX_DIM);
            B200_REQUIRE(a->data_type == B200WMMA_OUT_F16 || a->data_type == B200WMMA_OUT_BF16, B200WMMA_ERR_INVALID_ARG,
                         "%s: data_type must be B200WMMA_OUT_F16 or B200WMMA_OUT_BF16", who);
            B200_REQUIRE(a->scale - a->scale == 0.0f, B200WMMA_ERR_INVALID_ARG, "%s: scale must be finite", who);
            B200_REQUIRE(a->cap >= 0.0f && a->cap - a->cap == 0.0f, B200WMMA_ERR_INVALID_ARG,
                         "%s: cap must be finite and not negative (0 = none)", who);
            // constants made of them, 2 log2(e) scale / cap among them, have to be normal numbers
            const float limit = 1e30f, magnitude = a->scale < 0.0f ? -a->scale : a->scale;
            B200_REQUIRE(magnitude <= limit && (a->cap == 0.0f || (a->cap >= 1.0f / limit && a->cap <= limit && magnitude / a->cap <= limit)),
                         B200WMMA_ERR_UNSUPPORTED, "%s: scale, cap, 1 / cap and scale / cap must be at most 1e30", who);
            B200_REQUIRE(a->cap == 0.0f || magnitude == 0.0f || magnitude / a->cap >= 1e-37f, B200WMMA_ERR_UNSUPPORTED,
                         "%s: scale / cap must be 0 or at least 1e-37", who);
            return B200WMMA_OK;
        }
    } // namespace attn
} // namespace b200wmma
